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
  uint32_t site, step;
  uint32_t cut;     // threshold << 16, what a 16-bit value in the high half of a word has to reach
  uint32_t none;    // threshold 65536: nothing is kept
  float scale;
};

inline DropSpec drop_spec(const advopt_dropout_spec& s) {
  DropSpec d;
  d.keys = philox_keys(s.seed);
  d.step_dev = s.step_dev;
  d.site = s.site;
  d.step = s.step;
  d.none = s.threshold > 65535u;
  d.cut = d.none ? 0xFFFFFFFFu : s.threshold << 16;
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

// The 16-bit values of elements k0 .. k0 + 7, two per word.  k0 a multiple of 8
// takes one evaluation, other starts two.
__device__ __forceinline__ U4 drop_values(const DropSpec& d, uint32_t step, uint64_t k0) {
  const U4 w = drop_group(d, step, k0 >> 3);
  const uint32_t off = (uint32_t)(k0 & 7);
  if (off == 0) return w;
  // shift the two groups' 256 bits down by off 16-bit values: by 4, 2 and 1 of them
  const U4 x = drop_group(d, step, (k0 >> 3) + 1);
  const bool by4 = off & 4, by2 = off & 2, by1 = off & 1;
  const uint32_t s0 = by4 ? w.z : w.x, s1 = by4 ? w.w : w.y, s2 = by4 ? x.x : w.z, s3 = by4 ? x.y : w.w,
                 s4 = by4 ? x.z : x.x, s5 = by4 ? x.w : x.y;
  const uint32_t t[5] = {by2 ? s1 : s0, by2 ? s2 : s1, by2 ? s3 : s2, by2 ? s4 : s3, by2 ? s5 : s4};
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = by1 ? __funnelshift_r(t[i], t[i + 1], 16) : t[i];
  return U4{r[0], r[1], r[2], r[3]};
}

// v[e] of elements k0 + e becomes v[e] * scale where the element is kept, else
// 0.  The odd elements' values are compared where they lie, in the words' high
// halves.
__device__ __forceinline__ void drop8(float (&v)[8], const DropSpec& d, uint32_t step, uint64_t k0) {
  if (d.none) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    return;
  }
  const U4 w = drop_values(d, step, k0);
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __fmul_rn(v[2 * i], d.scale), b = __fmul_rn(v[2 * i + 1], d.scale);
    v[2 * i] = (q[i] << 16) >= d.cut ? a : 0.0f;
    v[2 * i + 1] = q[i] >= d.cut ? b : 0.0f;
  }
}

// Which of elements k0 .. k0 + 7 are kept, a bit each.
__device__ __forceinline__ uint32_t drop_bits8(const DropSpec& d, uint32_t step, uint64_t k0) {
  if (d.none) return 0u;
  const U4 w = drop_values(d, step, k0);
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= ((q[i] << 16) >= d.cut ? 1u << (2 * i) : 0u) | (q[i] >= d.cut ? 2u << (2 * i) : 0u);
  return bits;
}

// The same as drop8 on packed bf16 pairs, without the scale: dropped halves become 0.
__device__ __forceinline__ void drop_packed(uint32_t (&v)[4], const DropSpec& d, uint32_t step, uint64_t k0) {
  if (d.none) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0u;
    return;
  }
  const U4 w = drop_values(d, step, k0);
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] &= ((q[i] << 16) >= d.cut ? 0x0000FFFFu : 0u) | (q[i] >= d.cut ? 0xFFFF0000u : 0u);
}

__device__ __forceinline__ float drop1(float v, const DropSpec& d, uint32_t step, uint64_t k) {
  const uint32_t i = (uint32_t)(k & 7);
  const uint32_t w = drop_word(drop_group(d, step, k >> 3), i >> 1);
  return !d.none && ((i & 1) ? w : w << 16) >= d.cut ? __fmul_rn(v, d.scale) : 0.0f;
}

// Two bf16 values, the first in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Argument checks of a spec; nullptr when it is fine.
inline const char* drop_check(const advopt_dropout_spec& s) {
  if (s.threshold > 65536u) return "dropout: the threshold is at most 65536";
  if (reinterpret_cast<uintptr_t>(s.step_dev) & 7) return "dropout: step_dev must be 8-byte aligned";
  return nullptr;
}

}  // namespace advopt
