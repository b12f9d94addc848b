// Policy and preference losses over tokens' log-probabilities.
//
// Both are a masked sum over tokens, a little arithmetic on the sums, and a
// gradient that is elementwise in what the sums gave.  Bound by HBM for large
// batches and by the launches for small ones.  A warp takes up to 1024 tokens
// of a row and leaves its float32 sums; they are added in float64, in order,
// by one CTA, which is the same one where there are few: results repeat bit
// for bit.
#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace advopt {
namespace loss {

constexpr int64_t UNIT = 1024;           // tokens of a warp
constexpr int64_t ONE_CTA = 64;          // units that one CTA does alone
constexpr int FINISH = 1024;             // threads of the CTA that adds up

template <bool BF16>
__device__ __forceinline__ float get(const void* p, int64_t k) {
  return BF16 ? bf16_to_f(__ldg(static_cast<const uint16_t*>(p) + k)) : __ldg(static_cast<const float*>(p) + k);
}
template <bool BF16>
__device__ __forceinline__ void put(void* p, int64_t k, float v) {
  if (BF16) static_cast<uint16_t*>(p)[k] = (uint16_t)f_to_bf16_rne(v);
  else static_cast<float*>(p)[k] = v;
}

// Sums of N doubles over the CTA (FINISH threads), for thread 0.
template <int N>
__device__ __forceinline__ void cta_sum(double (&v)[N], double (*red)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_d(v[i]);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.x >> 5][i] = v[i];
  }
  __syncthreads();
  if (threadIdx.x < 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum_d(red[threadIdx.x][i]);
  }
}

// e^q - q - 1 without the cancellation near 0: there the series q^2 (1/2 + q/6
// + q^2/24 + ..), cut where the next term is below 2^-24 of the sum at |q| = 1/2.
__device__ __forceinline__ float kl_of(float q, float e1) {
  if (fabsf(q) > 0.5f) return __fsub_rn(e1, q);
  float p = 1.0f / 3628800.0f;
  p = __fmaf_rn(p, q, 1.0f / 362880.0f);
  p = __fmaf_rn(p, q, 1.0f / 40320.0f);
  p = __fmaf_rn(p, q, 1.0f / 5040.0f);
  p = __fmaf_rn(p, q, 1.0f / 720.0f);
  p = __fmaf_rn(p, q, 1.0f / 120.0f);
  p = __fmaf_rn(p, q, 1.0f / 24.0f);
  p = __fmaf_rn(p, q, 1.0f / 6.0f);
  p = __fmaf_rn(p, q, 0.5f);
  return __fmul_rn(__fmul_rn(q, q), p);
}

// ---- the policy loss ----
// A unit's sums: {kl_weight kl - gain, kl, clipped, tokens}.
template <bool BF16>
__device__ __forceinline__ float4 policy_unit(const advopt_policy_loss_args& a, int64_t r, int64_t c0) {
  const int lane = threadIdx.x & 31;
  const int64_t end = a.cols < c0 + UNIT ? a.cols : c0 + UNIT;
  const float row_adv = a.ld_adv < 0 ? get<BF16>(a.advantages, r) : 0.0f;
  const float high = __fadd_rn(1.0f, a.clip_high), low = __fsub_rn(1.0f, a.clip_low);
  float loss = 0.0f, kls = 0.0f, clips = 0.0f, count = 0.0f;
#pragma unroll 4
  for (int64_t c = c0 + lane; c < end; c += 32) {
    float slope = 0.0f;
    if (!a.mask || a.mask[r * a.ld_mask + c]) {
      const float p = get<BF16>(a.logprobs, r * a.ld_logprobs + c), old = get<BF16>(a.old, r * a.ld_old + c);
      const float adv = a.ld_adv < 0 ? row_adv : get<BF16>(a.advantages, r * a.ld_adv + c);
      // the clipping is decided in float64, where the difference is exact or nearly so
      const double d = (double)p - (double)old;
      const bool clipped = adv > 0.0f ? d > a.log_high : adv < 0.0f && d < a.log_low;
      float gain;
      if (clipped) {
        gain = __fmul_rn(adv > 0.0f ? high : low, adv);
      } else {
        gain = __fmul_rn(expf((float)d), adv);
        slope = -gain;
      }
      float kl = 0.0f;
      if (a.ref) {
        const float q = __fsub_rn(get<BF16>(a.ref, r * a.ld_ref + c), p), e1 = expm1f(q);
        kl = kl_of(q, e1);
        slope = __fmaf_rn(-a.kl_weight, e1, slope);
      }
      loss = __fadd_rn(loss, __fmaf_rn(a.kl_weight, kl, -gain));
      kls = __fadd_rn(kls, kl);
      clips += clipped ? 1.0f : 0.0f;
      count += 1.0f;
    }
    if (a.slope) a.slope[r * a.cols + c] = slope;
  }
  return make_float4(warp_sum(loss), warp_sum(kls), warp_sum(clips), warp_sum(count));
}

__device__ __forceinline__ void policy_finish(const advopt_policy_loss_args& a, int64_t per_row) {
  __shared__ double red[32][5];
  __shared__ double share;
  const float4* unit = static_cast<const float4*>(a.work);
  double t[5] = {};   // loss, kl, clipped, tokens, rows with a token
  for (int64_t r = threadIdx.x; r < a.rows; r += FINISH) {
    double row[4] = {};
    for (int64_t k = 0; k < per_row; ++k) {
      const float4 u = unit[r * per_row + k];
      row[0] += u.x; row[1] += u.y; row[2] += u.z; row[3] += u.w;
    }
    t[0] += !a.by_rows ? row[0] : row[3] > 0.0 ? row[0] / row[3] : 0.0;
    t[1] += row[1];
    t[2] += row[2];
    t[3] += row[3];
    t[4] += row[3] > 0.0 ? 1.0 : 0.0;
    a.scale[r] = row[3] > 0.0 ? (float)(1.0 / row[3]) : 0.0f;   // by rows: times 1 / rows below
  }
  cta_sum<5>(t, red);
  if (threadIdx.x == 0) {
    const double tokens = t[3] > 0.0 ? t[3] : 1.0;
    share = 1.0 / (a.by_rows ? (t[4] > 0.0 ? t[4] : 1.0) : tokens);
    *a.loss = (float)(t[0] * share);
    *a.kl = (float)(t[1] / tokens);
    *a.clipped = (float)(t[2] / tokens);
  }
  __syncthreads();
  const float s = (float)share;
  for (int64_t r = threadIdx.x; r < a.rows; r += FINISH) a.scale[r] = a.by_rows ? __fmul_rn(a.scale[r], s) : s;
}

template <bool BF16>
__device__ __forceinline__ void policy_units(const advopt_policy_loss_args& a, int64_t per_row, int64_t first, int64_t step) {
  for (int64_t u = first; u < a.rows * per_row; u += step) {
    const int64_t r = u / per_row;
    const float4 v = policy_unit<BF16>(a, r, (u - r * per_row) * UNIT);
    if ((threadIdx.x & 31) == 0) static_cast<float4*>(a.work)[u] = v;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256) policy_kernel(const __grid_constant__ advopt_policy_loss_args a, int64_t per_row) {
  policy_units<BF16>(a, per_row, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (int64_t)gridDim.x * 8);
}
__global__ void __launch_bounds__(FINISH) policy_finish_kernel(const __grid_constant__ advopt_policy_loss_args a, int64_t per_row) {
  policy_finish(a, per_row);
}
template <bool BF16>
__global__ void __launch_bounds__(FINISH) policy_one_kernel(const __grid_constant__ advopt_policy_loss_args a, int64_t per_row) {
  policy_units<BF16>(a, per_row, threadIdx.x >> 5, FINISH / 32);
  __syncthreads();
  policy_finish(a, per_row);
}

// A zero slope stays one, whatever the factors: a masked token's gradient is 0.
template <bool BF16>
__global__ void __launch_bounds__(256) policy_grad_kernel(void* out, const float* dloss, const float* slope, const float* scale, int64_t rows,
                                                          int64_t cols, int64_t per_row) {
  const float d = *dloss;
  const int lane = threadIdx.x & 31;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * per_row; u += (int64_t)gridDim.x * 8) {
    const int64_t r = u / per_row, c0 = (u - r * per_row) * UNIT, end = cols < c0 + UNIT ? cols : c0 + UNIT;
    const float k = __fmul_rn(d, scale[r]);
#pragma unroll 4
    for (int64_t c = c0 + lane; c < end; c += 32) {
      const float v = __ldg(slope + r * cols + c);
      put<BF16>(out, r * cols + c, v == 0.0f ? 0.0f : __fmul_rn(k, v));
    }
  }
}

// ---- the preference loss ----
template <bool BF16>
__device__ __forceinline__ float2 preference_unit(const advopt_preference_loss_args& a, int64_t r, int64_t c0) {
  const int64_t end = a.cols < c0 + UNIT ? a.cols : c0 + UNIT;
  float sum = 0.0f, count = 0.0f;
#pragma unroll 4
  for (int64_t c = c0 + (threadIdx.x & 31); c < end; c += 32)
    if (!a.mask || a.mask[r * a.ld_mask + c]) {
      const float p = get<BF16>(a.logprobs, r * a.ld_logprobs + c);
      sum = __fadd_rn(sum, a.ref ? __fsub_rn(p, get<BF16>(a.ref, r * a.ld_ref + c)) : p);
      count += 1.0f;
    }
  return make_float2(warp_sum(sum), warp_sum(count));
}

__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

__device__ __forceinline__ void preference_finish(const advopt_preference_loss_args& a, int64_t per_row) {
  __shared__ double red[32][1];
  const float2* unit = static_cast<const float2*>(a.work);
  double t[1] = {};
  for (int64_t i = threadIdx.x; i < a.pairs; i += FINISH) {
    double s[2], n[2];
    for (int k = 0; k < 2; ++k) {
      const int64_t r = i + k * a.pairs;
      double sum = 0.0, count = 0.0;
      for (int64_t j = 0; j < per_row; ++j) {
        sum += unit[r * per_row + j].x;
        count += unit[r * per_row + j].y;
      }
      n[k] = a.average && count > 0.0 ? count : 1.0;
      s[k] = (double)a.beta * (sum / n[k]);
      a.rewards[r] = (float)s[k];
    }
    const double h = s[0] - s[1], e = a.smoothing;
    t[0] += (1.0 - e) * softplus(-h) + e * softplus(h);
    if (a.slope) {
      const double k = (double)a.beta / (double)a.pairs * (e - 1.0 / (1.0 + exp(h)));   // -(1 - e) sig(-h) + e sig(h)
      a.slope[i] = (float)(k / n[0]);
      a.slope[i + a.pairs] = (float)(-k / n[1]);
    }
  }
  cta_sum<1>(t, red);
  if (threadIdx.x == 0) *a.loss = (float)(t[0] / (double)a.pairs);
}

template <bool BF16>
__device__ __forceinline__ void preference_units(const advopt_preference_loss_args& a, int64_t per_row, int64_t first, int64_t step) {
  for (int64_t u = first; u < 2 * a.pairs * per_row; u += step) {
    const int64_t r = u / per_row;
    const float2 v = preference_unit<BF16>(a, r, (u - r * per_row) * UNIT);
    if ((threadIdx.x & 31) == 0) static_cast<float2*>(a.work)[u] = v;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256) preference_kernel(const __grid_constant__ advopt_preference_loss_args a, int64_t per_row) {
  preference_units<BF16>(a, per_row, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (int64_t)gridDim.x * 8);
}
__global__ void __launch_bounds__(FINISH) preference_finish_kernel(const __grid_constant__ advopt_preference_loss_args a, int64_t per_row) {
  preference_finish(a, per_row);
}
template <bool BF16>
__global__ void __launch_bounds__(FINISH) preference_one_kernel(const __grid_constant__ advopt_preference_loss_args a, int64_t per_row) {
  preference_units<BF16>(a, per_row, threadIdx.x >> 5, FINISH / 32);
  __syncthreads();
  preference_finish(a, per_row);
}

template <bool BF16>
__global__ void __launch_bounds__(256) preference_grad_kernel(void* out, const float* dloss, const float* slope, const uint8_t* mask, int64_t ld_mask,
                                                              int64_t rows, int64_t cols, int64_t per_row) {
  const float d = *dloss;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * per_row; u += (int64_t)gridDim.x * 8) {
    const int64_t r = u / per_row, c0 = (u - r * per_row) * UNIT, end = cols < c0 + UNIT ? cols : c0 + UNIT;
    const float k = __fmul_rn(d, slope[r]);
#pragma unroll 4
    for (int64_t c = c0 + (threadIdx.x & 31); c < end; c += 32) put<BF16>(out, r * cols + c, !mask || mask[r * ld_mask + c] ? k : 0.0f);
  }
}

inline unsigned grid_of(int64_t units) {
  const int64_t ctas = ceil_div(units, 8);
  return (unsigned)(ctas < 148 * 32 ? ctas : 148 * 32);
}
inline bool sizes_ok(int64_t rows, int64_t cols) {
  return rows >= 0 && cols >= 0 && rows < (int64_t)1 << 31 && cols < (int64_t)1 << 31 && (cols == 0 || rows <= ((int64_t)1 << 46) / cols);
}
inline bool pitch_ok(int64_t ld, int64_t rows, int64_t cols) { return rows <= 1 || ld >= cols; }

}  // namespace loss
}  // namespace advopt

using namespace advopt;

extern "C" int64_t advopt_policy_loss_work(int64_t rows, int64_t cols) {
  return rows <= 0 ? 0 : rows * ceil_div(cols > 0 ? cols : 0, loss::UNIT) * 16;
}

extern "C" int advopt_policy_loss(const advopt_policy_loss_args* a, void* stream) {
  if (!a || !loss::sizes_ok(a->rows, a->cols) || !a->loss || !a->kl || !a->clipped || !(a->clip_low >= 0.0f && a->clip_low <= 1.0f) || !(a->clip_high >= 0.0f) ||
      !(a->kl_weight - a->kl_weight == 0.0f))
    return set_error(ADVOPT_E_INVALID, "advopt_policy_loss: bad arguments");
  if (!known_dtype(a->dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_policy_loss: float32 and bfloat16 are supported");
  const bool any = a->rows && a->cols;
  if (any && (!a->scale || !a->logprobs || !a->old || !a->advantages || !a->work || !aligned16(a->work) ||
              !loss::pitch_ok(a->ld_logprobs, a->rows, a->cols) || !loss::pitch_ok(a->ld_old, a->rows, a->cols) ||
              (a->ref && !loss::pitch_ok(a->ld_ref, a->rows, a->cols)) || (a->mask && !loss::pitch_ok(a->ld_mask, a->rows, a->cols)) ||
              (a->ld_adv >= 0 && !loss::pitch_ok(a->ld_adv, a->rows, a->cols))))
    return set_error(ADVOPT_E_INVALID, "advopt_policy_loss: null or unaligned pointer, or a pitch below the row's length");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  advopt_policy_loss_args q = *a;
  if (!any) q.rows = 0;
  const int64_t per_row = ceil_div(a->cols, loss::UNIT), units = q.rows * per_row;
  const bool bf16 = a->dtype == ADVOPT_DT_BF16;
  if (units <= loss::ONE_CTA) {
    if (bf16) loss::policy_one_kernel<true><<<1, loss::FINISH, 0, s>>>(q, per_row);
    else loss::policy_one_kernel<false><<<1, loss::FINISH, 0, s>>>(q, per_row);
  } else {
    if (bf16) loss::policy_kernel<true><<<loss::grid_of(units), 256, 0, s>>>(q, per_row);
    else loss::policy_kernel<false><<<loss::grid_of(units), 256, 0, s>>>(q, per_row);
    loss::policy_finish_kernel<<<1, loss::FINISH, 0, s>>>(q, per_row);
  }
  return check_cuda(cudaGetLastError(), "advopt_policy_loss");
}

extern "C" int advopt_policy_loss_grad(void* out, const float* dloss, const float* slope, const float* scale, int64_t rows, int64_t cols,
                                       int32_t dtype, void* stream) {
  if (!loss::sizes_ok(rows, cols)) return set_error(ADVOPT_E_INVALID, "advopt_policy_loss_grad: bad arguments");
  if (!known_dtype(dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_policy_loss_grad: float32 and bfloat16 are supported");
  if (rows == 0 || cols == 0) return ADVOPT_OK;
  if (!out || !dloss || !slope || !scale) return set_error(ADVOPT_E_INVALID, "advopt_policy_loss_grad: null pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t per_row = ceil_div(cols, loss::UNIT);
  const unsigned grid = loss::grid_of(rows * per_row);
  if (dtype == ADVOPT_DT_BF16) loss::policy_grad_kernel<true><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  else loss::policy_grad_kernel<false><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  return check_cuda(cudaGetLastError(), "advopt_policy_loss_grad");
}

extern "C" int64_t advopt_preference_loss_work(int64_t pairs, int64_t cols) {
  return pairs <= 0 ? 0 : 2 * pairs * ceil_div(cols > 0 ? cols : 0, loss::UNIT) * 8;
}

extern "C" int advopt_preference_loss(const advopt_preference_loss_args* a, void* stream) {
  if (!a || a->pairs < 1 || a->pairs >= (int64_t)1 << 30 || !loss::sizes_ok(2 * a->pairs, a->cols) || !a->loss || !a->rewards ||
      !(a->beta - a->beta == 0.0f) || !(a->smoothing >= 0.0f && a->smoothing <= 1.0f))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss: bad arguments");
  if (!known_dtype(a->dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_preference_loss: float32 and bfloat16 are supported");
  const int64_t rows = 2 * a->pairs;
  if (a->cols && (!a->logprobs || !a->work || !aligned16(a->work) || !loss::pitch_ok(a->ld_logprobs, rows, a->cols) ||
                  (a->ref && !loss::pitch_ok(a->ld_ref, rows, a->cols)) || (a->mask && !loss::pitch_ok(a->ld_mask, rows, a->cols))))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss: null or unaligned pointer, or a pitch below the row's length");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t per_row = ceil_div(a->cols, loss::UNIT), units = rows * per_row;
  const bool bf16 = a->dtype == ADVOPT_DT_BF16;
  if (units <= loss::ONE_CTA) {
    if (bf16) loss::preference_one_kernel<true><<<1, loss::FINISH, 0, s>>>(*a, per_row);
    else loss::preference_one_kernel<false><<<1, loss::FINISH, 0, s>>>(*a, per_row);
  } else {
    if (bf16) loss::preference_kernel<true><<<loss::grid_of(units), 256, 0, s>>>(*a, per_row);
    else loss::preference_kernel<false><<<loss::grid_of(units), 256, 0, s>>>(*a, per_row);
    loss::preference_finish_kernel<<<1, loss::FINISH, 0, s>>>(*a, per_row);
  }
  return check_cuda(cudaGetLastError(), "advopt_preference_loss");
}

extern "C" int advopt_preference_loss_grad(void* out, const float* dloss, const float* slope, const uint8_t* mask, int64_t ld_mask, int64_t pairs,
                                           int64_t cols, int32_t dtype, void* stream) {
  if (pairs < 0 || pairs >= (int64_t)1 << 30 || !loss::sizes_ok(2 * pairs, cols))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss_grad: bad arguments");
  if (!known_dtype(dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_preference_loss_grad: float32 and bfloat16 are supported");
  if (pairs == 0 || cols == 0) return ADVOPT_OK;
  if (!out || !dloss || !slope || (mask && !loss::pitch_ok(ld_mask, 2 * pairs, cols)))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss_grad: null pointer or a pitch below the row's length");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t per_row = ceil_div(cols, loss::UNIT);
  const unsigned grid = loss::grid_of(2 * pairs * per_row);
  if (dtype == ADVOPT_DT_BF16) loss::preference_grad_kernel<true><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, 2 * pairs, cols, per_row);
  else loss::preference_grad_kernel<false><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, 2 * pairs, cols, per_row);
  return check_cuda(cudaGetLastError(), "advopt_preference_loss_grad");
}
