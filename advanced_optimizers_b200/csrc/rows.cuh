// Eight consecutive elements of a row, kept as they lie in memory (bf16 ones
// packed: half the registers), shared by the kernels that work on rows.
#pragma once

#include "common.cuh"
#include "drop.cuh"

namespace advopt {

template <bool BF16>
struct Oct {
  static constexpr int kBytes = BF16 ? 2 : 4;
  static constexpr int kWords = BF16 ? 4 : 8;
  uint32_t w[kWords];

  __device__ __forceinline__ float at(int e) const {
    if (!BF16) return u2f(w[BF16 ? 0 : e]);
    return u2f((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
  }
  // Elements 2i and 2i + 1.
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(at(2 * i), at(2 * i + 1)); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  // 16-byte aligned, through the read-only path.
  __device__ __forceinline__ void load(const void* base, int64_t k) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + k * kBytes);
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 q = __ldg(p + i);
      w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
    }
  }
  // The first nv elements one by one, zeros behind them.
  __device__ __forceinline__ void load_some(const void* base, int64_t k, int nv) {
    if (BF16) {
      const uint16_t* p = static_cast<const uint16_t*>(base) + k;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        w[i] = (2 * i < nv ? (uint32_t)__ldg(p + 2 * i) : 0u) | (2 * i + 1 < nv ? (uint32_t)__ldg(p + 2 * i + 1) << 16 : 0u);
    } else {
      const uint32_t* p = static_cast<const uint32_t*>(base) + k;
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = i < nv ? __ldg(p + i) : 0u;
    }
  }
  __device__ __forceinline__ void get(const void* base, int64_t k, int nv, bool vec) {
    if (vec && nv == 8) load(base, k);
    else load_some(base, k, nv);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = BF16 ? bf16x2(v[2 * (i & 3)], v[2 * (i & 3) + 1]) : f2u(v[i]);
  }
  __device__ __forceinline__ void store(void* base, int64_t k) const {
    uint4* p = reinterpret_cast<uint4*>(static_cast<unsigned char*>(base) + k * kBytes);
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) p[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  __device__ __forceinline__ void store_some(void* base, int64_t k, int nv) const {
    if (BF16) {
      uint16_t* p = static_cast<uint16_t*>(base) + k;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < nv) p[e] = (uint16_t)(w[(e >> 1) & (kWords - 1)] >> (16 * (e & 1)));
    } else {
      uint32_t* p = static_cast<uint32_t*>(base) + k;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < nv) p[e] = w[e & (kWords - 1)];
    }
  }
  __device__ __forceinline__ void put(void* base, int64_t k, int nv, bool vec) const {
    if (vec && nv == 8) store(base, k);
    else store_some(base, k, nv);
  }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int bytes_of(int dtype) { return dtype == ADVOPT_DT_BF16 ? 2 : 4; }
inline bool known_dtype(int dtype) { return dtype == ADVOPT_DT_F32 || dtype == ADVOPT_DT_BF16; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace advopt
