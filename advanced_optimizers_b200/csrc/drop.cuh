// Counter-based dropout shared by the dropout kernel, the fp8 quantiser and
// the fp8 GEMM's epilogue: element k of a tensor is kept iff its 16-bit
// Philox value (stream kNoiseDrop, the mapping of philox_u16x8) reaches the
// threshold, so every kernel that touches element k finds the same mask
// without one being stored.  16 bits per element: one Philox evaluation (20
// wide multiplies) serves eight elements, which a bf16 pass hides under its
// memory time; p is realised in steps of 2^-16 and the scale is the inverse
// of the realised probability, so the expectation is exact.
#pragma once

#include "advopt.h"
#include "common.cuh"

namespace advopt {

struct DropSpec {
  PhiloxKeys keys;
  const int64_t* step_dev;
  uint32_t site, step, threshold;
  float scale;
};

inline DropSpec drop_spec(const advopt_dropout_spec& s) {
  DropSpec d;
  d.keys = philox_keys(s.seed);
  d.step_dev = s.step_dev;
  d.site = s.site;
  d.step = s.step;
  d.threshold = s.threshold;
  d.scale = s.scale;
  return d;
}

// The step of a launch: a host value, or read where a captured graph's replay finds it.
__device__ __forceinline__ uint32_t drop_step(const DropSpec& d) {
  return d.step_dev ? (uint32_t)__ldg(reinterpret_cast<const unsigned long long*>(d.step_dev)) : d.step;
}

// The eight 16-bit values of group `grp` (elements 8 grp .. 8 grp + 7), two per word.
__device__ __forceinline__ U4 drop_group(const DropSpec& d, uint32_t step, uint64_t grp) {
  return philox4x32_10_k(
      U4{(uint32_t)grp, (uint32_t)(grp >> 32) | ((uint32_t)kNoiseDrop << 24), d.site, step}, d.keys);
}

__device__ __forceinline__ uint32_t drop_word(const U4& w, uint32_t i) {
  return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
}

// keep bits (bit e: element k0 + e) of N consecutive elements, N a multiple
// of 4 up to 16.  k0 a multiple of 8 takes N / 8 evaluations; other starts
// evaluate each group they touch.
template <int N>
__device__ __forceinline__ uint32_t drop_keep(const DropSpec& d, uint32_t step, uint64_t k0) {
  uint32_t bits = 0;
  if (N >= 8 && (k0 & 7) == 0) {
#pragma unroll
    for (int g = 0; g < N / 8; ++g) {
      const U4 w = drop_group(d, step, (k0 >> 3) + g);
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t r = (e & 1) ? q[e >> 1] >> 16 : q[e >> 1] & 0xFFFFu;
        bits |= (r >= d.threshold ? 1u : 0u) << (8 * g + e);
      }
    }
    return bits;
  }
  int e = 0;
#pragma unroll 1
  for (uint64_t grp = k0 >> 3; e < N; ++grp) {
    const U4 w = drop_group(d, step, grp);
#pragma unroll 1
    for (uint32_t i = (uint32_t)((k0 + e) & 7); i < 8 && e < N; ++i, ++e) {
      const uint32_t r = (drop_word(w, i >> 1) >> (16 * (i & 1))) & 0xFFFFu;
      bits |= (r >= d.threshold ? 1u : 0u) << e;
    }
  }
  return bits;
}

__device__ __forceinline__ bool drop_keep1(const DropSpec& d, uint32_t step, uint64_t k) {
  const uint32_t i = (uint32_t)(k & 7);
  return ((drop_word(drop_group(d, step, k >> 3), i >> 1) >> (16 * (i & 1))) & 0xFFFFu) >= d.threshold;
}

// Argument checks of a spec; nullptr when it is fine.
inline const char* drop_check(const advopt_dropout_spec& s) {
  if (s.threshold > 65536u) return "dropout: the threshold is at most 65536";
  if (reinterpret_cast<uintptr_t>(s.step_dev) & 7) return "dropout: step_dev must be 8-byte aligned";
  return nullptr;
}

}  // namespace advopt
