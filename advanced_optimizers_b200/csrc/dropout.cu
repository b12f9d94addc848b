// y = residual + keep * x * scale with the mask drawn on the fly (drop.cuh).
//
// Bound: HBM.  bf16 with a residual moves 6 bytes per element; the Philox
// rounds are 2.5 wide multiplies per element.
#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "drop.cuh"

namespace advopt {
namespace {

__host__ __device__ constexpr int groups_a_trip(bool bf16, bool res) { return bf16 && !res ? 4 : 2; }

template <bool BF16>
struct Raw {
  uint4 w[BF16 ? 1 : 2];   // eight elements as they lie in memory
  template <bool IN_PLACE>
  __device__ __forceinline__ void load(const void* base, int64_t k0) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + k0 * (BF16 ? 2 : 4));
#pragma unroll
    for (int i = 0; i < (BF16 ? 1 : 2); ++i) w[i] = IN_PLACE ? p[i] : __ldg(p + i);
  }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
    if (BF16) {
      const uint32_t q[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = u2f(q[i] << 16);
        v[2 * i + 1] = u2f(q[i] & 0xFFFF0000u);
      }
    } else {
      const uint4& h = w[BF16 ? 0 : 1];
      const uint32_t q[8] = {w[0].x, w[0].y, w[0].z, w[0].w, h.x, h.y, h.z, h.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = u2f(q[i]);
    }
  }
};

template <bool BF16, bool IN_PLACE>
__device__ __forceinline__ void load_group(const void* base, int64_t k0, int nv, bool vec, float (&v)[8]) {
  if (vec) {
    Raw<BF16> r;
    r.template load<IN_PLACE>(base, k0);
    r.floats(v);
  } else {
    load8<BF16>(base, k0, nv, false, v);   // element by element, plain loads
  }
}

template <bool BF16>
__device__ __forceinline__ void store_group(void* y, int64_t k0, int nv, bool vec, const float (&a)[8]) {
  if (BF16) {
    const uint32_t w[4] = {bf16x2(a[0], a[1]), bf16x2(a[2], a[3]), bf16x2(a[4], a[5]), bf16x2(a[6], a[7])};
    uint16_t* out = static_cast<uint16_t*>(y) + k0;
    if (vec) {
      *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < nv) out[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
  } else {
    store8_f32(y, k0, nv, vec, a);
  }
}

// U groups of eight elements a trip, a grid's width apart: all their loads are
// on their way before the first Philox evaluation.  One at a time, a bf16 pass
// had 24 KB in flight per SM and ran at 0.6 of HBM.
// IN_PLACE: y is x or res, whose loads may then not go through the read-only
// path (which lets a trip's loads pass the stores of the one before: 16384 x
// 4096 bf16 with a residual takes 62 us with it, 72 without).
template <bool BF16, bool RES, bool IN_PLACE>
__global__ void __launch_bounds__(256)
    dropout_kernel(void* y, const void* x, const void* res, int64_t n, bool vec, const __grid_constant__ DropSpec d) {
  constexpr int U = groups_a_trip(BF16, RES);
  const uint32_t step = drop_step(d);
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (vec) {
    for (; g + (U - 1) * stride < n >> 3; g += U * stride) {
      Raw<BF16> a[U], r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u].template load<IN_PLACE>(x, (g + u * stride) << 3);
        if (RES) r[u].template load<IN_PLACE>(res, (g + u * stride) << 3);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8], t[8];
        a[u].floats(v);
        drop8(v, d, step, (uint64_t)(g + u * stride) << 3);
        if (RES) {
          r[u].floats(t);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(t[e], v[e]);
        }
        store_group<BF16>(y, (g + u * stride) << 3, 8, true, v);
      }
    }
  }
  for (; g < (n + 7) >> 3; g += stride) {
    const int64_t k0 = g << 3;
    const int nv = n - k0 < 8 ? (int)(n - k0) : 8;
    const bool whole = vec && nv == 8;
    float v[8], t[8];
    load_group<BF16, IN_PLACE>(x, k0, nv, whole, v);
    if (RES) load_group<BF16, IN_PLACE>(res, k0, nv, whole, t);
    drop8(v, d, step, (uint64_t)k0);
    if (RES) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(t[e], v[e]);
    }
    store_group<BF16>(y, k0, nv, whole, v);
  }
}

template <bool BF16>
void launch(void* y, const void* x, const void* res, int64_t n, const DropSpec& d, cudaStream_t s) {
  const int64_t groups = (n + 7) >> 3, trip = 256 * groups_a_trip(BF16, res != nullptr);
  // whole trips for every thread where that still gives each SM two CTAs, else one group a thread
  const int64_t blocks = groups >= 2 * 148 * trip ? (groups + trip - 1) / trip : (groups + 255) / 256;
  const int grid = (int)(blocks < 148 * 8 ? blocks : 148 * 8);
  const bool vec = ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res)) & 15) == 0;
  const uintptr_t bytes = (uintptr_t)n * (BF16 ? 2 : 4), at = reinterpret_cast<uintptr_t>(y);
  const auto meets = [&](const void* p) {
    const uintptr_t q = reinterpret_cast<uintptr_t>(p);
    return p && q < at + bytes && at < q + bytes;
  };
  if (meets(x) || meets(res)) {
    if (res) dropout_kernel<BF16, true, true><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
    else dropout_kernel<BF16, false, true><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
  } else {
    if (res) dropout_kernel<BF16, true, false><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
    else dropout_kernel<BF16, false, false><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
  }
}

}  // namespace
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_dropout(void* y, const void* x, const void* residual, int64_t n, int32_t dtype,
                              const advopt_dropout_spec* spec, void* stream) {
  if (n < 0 || !spec || (n > 0 && (!x || !y))) return set_error(ADVOPT_E_INVALID, "advopt_dropout: bad arguments");
  if (dtype != ADVOPT_DT_F32 && dtype != ADVOPT_DT_BF16)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_dropout: float32 and bfloat16 tensors are supported");
  if (const char* why = drop_check(*spec)) return set_error(ADVOPT_E_INVALID, why);
  if (n == 0) return ADVOPT_OK;
  const DropSpec d = drop_spec(*spec);
  if (dtype == ADVOPT_DT_BF16) launch<true>(y, x, residual, n, d, static_cast<cudaStream_t>(stream));
  else launch<false>(y, x, residual, n, d, static_cast<cudaStream_t>(stream));
  return check_cuda(cudaGetLastError(), "advopt_dropout");
}
