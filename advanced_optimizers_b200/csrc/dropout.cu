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

template <bool BF16, bool RES>
__global__ void __launch_bounds__(256)
    dropout_kernel(void* y, const void* x, const void* res, int64_t n, bool vec, const __grid_constant__ DropSpec d) {
  const uint32_t step = drop_step(d);
  const int64_t groups = (n + 7) >> 3;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += stride) {
    const int64_t k0 = g << 3;
    const int nv = n - k0 < 8 ? (int)(n - k0) : 8;
    const bool v = vec && nv == 8;
    float a[8], r[8];
    load8<BF16>(x, k0, nv, v, a);
    if (RES) load8<BF16>(res, k0, nv, v, r);
    drop8(a, d, step, (uint64_t)k0);
    if (RES) {
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = __fadd_rn(r[e], a[e]);
    }
    if (BF16) {
      const uint32_t u[4] = {bf16x2(a[0], a[1]), bf16x2(a[2], a[3]), bf16x2(a[4], a[5]), bf16x2(a[6], a[7])};
      uint16_t* out = static_cast<uint16_t*>(y) + k0;
      if (v) {
        *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < nv) out[e] = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
      }
    } else {
      store8_f32(y, k0, nv, v, a);
    }
  }
}

template <bool BF16>
void launch(void* y, const void* x, const void* res, int64_t n, const DropSpec& d, cudaStream_t s) {
  const int64_t groups = (n + 7) >> 3;
  const int64_t blocks = (groups + 255) / 256;
  const int grid = (int)(blocks < 148 * 8 ? blocks : 148 * 8);
  const bool vec = ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res)) & 15) == 0;
  if (res) dropout_kernel<BF16, true><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
  else dropout_kernel<BF16, false><<<grid, 256, 0, s>>>(y, x, res, n, vec, d);
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
