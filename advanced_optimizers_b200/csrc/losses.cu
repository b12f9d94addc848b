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

constexpr int FINISH = 1024;             // threads of the CTA that adds up
constexpr int64_t BLOCK = 128;           // tokens that a warp takes at once, four a lane

// Tokens of a unit, which is a warp's: small ones, for many warps, until their
// sums are more than one CTA adds up in passing.
inline int64_t unit_of(int64_t rows, int64_t cols) { return rows * ceil_div(cols, BLOCK) <= 2048 ? BLOCK : 8 * BLOCK; }
constexpr int64_t GRAD_UNIT = 4 * BLOCK; // of the gradients' kernels
constexpr int64_t ONE_CTA = 128;         // units that one CTA does alone

// Four tokens of a lane: consecutive ones (VEC: aligned to four elements), or 32 apart.
template <bool BF16, bool VEC>
__device__ __forceinline__ void get4(float (&v)[4], const void* p, int64_t k, int64_t left) {
  const int lane = threadIdx.x & 31;
  if (VEC) {
    if (lane * 4 < left) {
      if (BF16) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + k) + lane);
        v[0] = u2f(q.x << 16); v[1] = u2f(q.x & 0xFFFF0000u); v[2] = u2f(q.y << 16); v[3] = u2f(q.y & 0xFFFF0000u);
      } else {
        const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + k) + lane);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left) {
        const int64_t at = k + lane + 32 * i;
        v[i] = BF16 ? bf16_to_f(__ldg(static_cast<const uint16_t*>(p) + at)) : __ldg(static_cast<const float*>(p) + at);
      }
  }
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void put4(void* p, int64_t k, int64_t left, const float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  if (VEC) {
    if (lane * 4 < left) {
      if (BF16) reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + k)[lane] = make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
      else reinterpret_cast<float4*>(static_cast<float*>(p) + k)[lane] = make_float4(v[0], v[1], v[2], v[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left) {
        const int64_t at = k + lane + 32 * i;
        if (BF16) static_cast<uint16_t*>(p)[at] = (uint16_t)f_to_bf16_rne(v[i]);
        else static_cast<float*>(p)[at] = v[i];
      }
  }
}
// Which of the four count, as bits.
template <bool VEC>
__device__ __forceinline__ uint32_t mask4(const uint8_t* p, int64_t k, int64_t left) {
  const int lane = threadIdx.x & 31;
  uint32_t on = 0;
  if (VEC) {
    if (lane * 4 < left) {
      const uint32_t q = p ? __ldg(reinterpret_cast<const uint32_t*>(p + k) + lane) : 0x01010101u;
#pragma unroll
      for (int i = 0; i < 4; ++i) on |= (q >> (8 * i) & 0xFFu) ? 1u << i : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < left && (!p || __ldg(p + k + lane + 32 * i))) on |= 1u << i;
  }
  return on;
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

// kl = e^q - q - 1 and e1 = e^q - 1.  Up to |q| = 1/2 by the series q^2 (1/2 +
// q/6 + q^2/24 + ..), without the cancellation near 0; the first term left out
// is below 2^-33 of the sum.
__device__ __forceinline__ void kl_of(float q, float& kl, float& e1) {
  if (fabsf(q) <= 0.5f) {
    float p = 1.0f / 3628800.0f;
    p = __fmaf_rn(p, q, 1.0f / 362880.0f);
    p = __fmaf_rn(p, q, 1.0f / 40320.0f);
    p = __fmaf_rn(p, q, 1.0f / 5040.0f);
    p = __fmaf_rn(p, q, 1.0f / 720.0f);
    p = __fmaf_rn(p, q, 1.0f / 120.0f);
    p = __fmaf_rn(p, q, 1.0f / 24.0f);
    p = __fmaf_rn(p, q, 1.0f / 6.0f);
    p = __fmaf_rn(p, q, 0.5f);
    kl = __fmul_rn(__fmul_rn(q, q), p);
    e1 = __fadd_rn(q, kl);
  } else {
    e1 = expm1f(q);
    kl = __fsub_rn(e1, q);
  }
}

// Whether p - old is above `border` (ABOVE) or below it.  The float32
// difference d is off by at most 2^-24 of itself and the rounded border by
// 2^-24: further apart than 2^-22 of the border the float32 comparison is
// right, nearer ones are compared in float64.
template <bool ABOVE>
__device__ __forceinline__ bool beyond(float p, float old, float d, double border, float border32) {
  if (fabsf(__fsub_rn(d, border32)) > __fmul_rn(0x1p-22f, fabsf(border32))) return ABOVE ? d > border32 : d < border32;
  const double e = (double)p - (double)old;
  return ABOVE ? e > border : e < border;
}

// e^d adv where e^d is about to leave float32 (e^88.7) or has: its root is a factor twice; an advantage of 0 stays 0 for any number d.
__device__ __forceinline__ float far_gain(float d, float adv) {
  const float root = expf(__fmul_rn(0.5f, d));
  return adv == 0.0f && d < __builtin_huge_valf() ? 0.0f : __fmul_rn(__fmul_rn(root, adv), root);
}

// ---- the policy loss ----
struct Policy {
  advopt_policy_loss_args a;
  int64_t per_row, unit;
  float high32, low32;      // the borders
};

// A unit's sums: {kl_weight kl - gain, kl, clipped, tokens}.
template <bool BF16, bool VEC>
__device__ __forceinline__ float4 policy_unit(const Policy& q, int64_t r, int64_t c0) {
  const advopt_policy_loss_args& a = q.a;
  const int64_t end = a.cols < c0 + q.unit ? a.cols : c0 + q.unit;
  const bool per_row = a.ld_adv < 0;
  const float row_adv = !per_row ? 0.0f : BF16 ? bf16_to_f(__ldg(static_cast<const uint16_t*>(a.advantages) + r))
                                               : __ldg(static_cast<const float*>(a.advantages) + r);
  const float high = __fadd_rn(1.0f, a.clip_high), low = __fsub_rn(1.0f, a.clip_low);
  float loss = 0.0f, kls = 0.0f, clips = 0.0f, count = 0.0f;
#pragma unroll 2
  for (int64_t c = c0; c < end; c += BLOCK) {
    const int64_t left = end - c;
    float p[4] = {}, old[4] = {}, ref[4] = {}, adv[4], slope[4] = {};
    const uint32_t on = mask4<VEC>(a.mask, r * a.ld_mask + c, left);
    get4<BF16, VEC>(p, a.logprobs, r * a.ld_logprobs + c, left);
    get4<BF16, VEC>(old, a.old, r * a.ld_old + c, left);
    if (a.ref) get4<BF16, VEC>(ref, a.ref, r * a.ld_ref + c, left);
#pragma unroll
    for (int i = 0; i < 4; ++i) adv[i] = row_adv;
    if (!per_row) get4<BF16, VEC>(adv, a.advantages, r * a.ld_adv + c, left);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!(on >> i & 1u)) continue;
      const float d = __fsub_rn(p[i], old[i]);
      const bool clipped = adv[i] > 0.0f ? beyond<true>(p[i], old[i], d, a.log_high, q.high32)
                                         : adv[i] < 0.0f && beyond<false>(p[i], old[i], d, a.log_low, q.low32);
      const float gain = d > 88.0f && !clipped ? far_gain(d, adv[i])   // a branch that hardly any warp takes: selects cost 29.7 us where it costs 28.4
                                               : __fmul_rn(clipped ? adv[i] > 0.0f ? high : low : expf(d), adv[i]);
      slope[i] = clipped ? 0.0f : -gain;
      float kl = 0.0f, e1;
      if (a.ref) {
        kl_of(__fsub_rn(ref[i], p[i]), kl, e1);
        if (a.kl_weight != 0.0f) slope[i] = __fmaf_rn(-a.kl_weight, e1, slope[i]);   // else kl is reported alone, and may be infinite
      }
      loss = __fadd_rn(loss, a.kl_weight != 0.0f ? __fmaf_rn(a.kl_weight, kl, -gain) : -gain);
      kls = __fadd_rn(kls, kl);
      clips += clipped ? 1.0f : 0.0f;
      count += 1.0f;
    }
    if (a.slope) put4<false, VEC>(a.slope, r * a.cols + c, left, slope);
  }
  return make_float4(warp_sum(loss), warp_sum(kls), warp_sum(clips), warp_sum(count));
}

// What the CTA's threads add to the sums of a row or of all tokens: the units
// of a row by one thread where they are few, else by a warp.
template <int N, class Unit, class Row>
__device__ __forceinline__ void each_row(int64_t rows, int64_t per_row, const Unit& unit, const Row& row) {
  if (per_row < 32) {
    for (int64_t r = threadIdx.x; r < rows; r += FINISH) {
      double s[N] = {};
      for (int64_t k = 0; k < per_row; ++k) unit(s, r * per_row + k);
      row(r, s);
    }
  } else {
    for (int64_t r = threadIdx.x >> 5; r < rows; r += FINISH / 32) {
      double s[N] = {};
      for (int64_t k = threadIdx.x & 31; k < per_row; k += 32) unit(s, r * per_row + k);
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = warp_sum_d(s[i]);
      if ((threadIdx.x & 31) == 0) row(r, s);
    }
  }
}

__device__ __forceinline__ void policy_finish(const Policy& q) {
  const advopt_policy_loss_args& a = q.a;
  __shared__ double red[32][5];
  __shared__ float share;
  const float4* units = static_cast<const float4*>(a.work);
  double t[5] = {};   // loss, kl, clipped, tokens, rows with a token
  const auto unit = [&](double (&s)[4], int64_t u) {
    const float4 v = units[u];
    s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
  };
  if (a.by_rows) {
    each_row<4>(a.rows, q.per_row, unit, [&](int64_t r, const double (&s)[4]) {
      const float n = (float)s[3];
      t[0] += n > 0.0f ? s[0] / s[3] : 0.0;
      t[1] += s[1]; t[2] += s[2]; t[3] += s[3];
      t[4] += n > 0.0f ? 1.0 : 0.0;
      a.scale[r] = n > 0.0f ? __fdiv_rn(1.0f, n) : 0.0f;   // times 1 / rows below
    });
  } else {
    double s[4] = {};
    for (int64_t u = threadIdx.x; u < a.rows * q.per_row; u += FINISH) unit(s, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = s[i];
  }
  cta_sum<5>(t, red);
  if (threadIdx.x == 0) {
    const double tokens = t[3] > 0.0 ? t[3] : 1.0, by = a.by_rows ? (t[4] > 0.0 ? t[4] : 1.0) : tokens;
    share = (float)(1.0 / by);
    *a.loss = (float)(t[0] / by);
    *a.kl = (float)(t[1] / tokens);
    *a.clipped = (float)(t[2] / tokens);
  }
  __syncthreads();
  const float s = share;
  for (int64_t r = threadIdx.x; r < a.rows; r += FINISH) a.scale[r] = a.by_rows ? __fmul_rn(a.scale[r], s) : s;
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void policy_units(const Policy& q, int64_t first, int64_t step) {
  for (int64_t u = first; u < q.a.rows * q.per_row; u += step) {
    const int64_t r = u / q.per_row;
    const float4 v = policy_unit<BF16, VEC>(q, r, (u - r * q.per_row) * q.unit);
    if ((threadIdx.x & 31) == 0) static_cast<float4*>(q.a.work)[u] = v;
  }
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) policy_kernel(const __grid_constant__ Policy q) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  policy_units<BF16, VEC>(q, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (int64_t)gridDim.x * 8);
}
__global__ void __launch_bounds__(FINISH) policy_finish_kernel(const __grid_constant__ Policy q) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  policy_finish(q);
}
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(FINISH) policy_one_kernel(const __grid_constant__ Policy q) {
  policy_units<BF16, VEC>(q, threadIdx.x >> 5, FINISH / 32);
  __syncthreads();
  policy_finish(q);
}

// A zero slope stays one, whatever the factors: a masked token's gradient is 0.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) policy_grad_kernel(void* out, const float* dloss, const float* slope, const float* scale, int64_t rows,
                                                          int64_t cols, int64_t per_row) {
  const float d = *dloss;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * per_row; u += (int64_t)gridDim.x * 8) {
    const int64_t r = u / per_row, c0 = (u - r * per_row) * GRAD_UNIT, end = cols < c0 + GRAD_UNIT ? cols : c0 + GRAD_UNIT;
    const float k = __fmul_rn(d, scale[r]);
#pragma unroll
    for (int j = 0; j < GRAD_UNIT / BLOCK; ++j) {
      const int64_t c = c0 + j * BLOCK;
      float v[4] = {};
      get4<false, VEC>(v, slope, r * cols + c, end - c);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = v[i] == 0.0f ? 0.0f : __fmul_rn(k, v[i]);
      put4<BF16, VEC>(out, r * cols + c, end - c, v);
    }
  }
}

// ---- the preference loss ----
struct Preference {
  advopt_preference_loss_args a;
  int64_t per_row, unit;
};

// A unit's sum of log ratios, and its tokens.
template <bool BF16, bool VEC>
__device__ __forceinline__ float2 preference_unit(const Preference& q, int64_t r, int64_t c0) {
  const advopt_preference_loss_args& a = q.a;
  const int64_t end = a.cols < c0 + q.unit ? a.cols : c0 + q.unit;
  float sum = 0.0f, count = 0.0f;
#pragma unroll 4
  for (int64_t c = c0; c < end; c += BLOCK) {
    const int64_t left = end - c;
    float p[4] = {}, ref[4] = {};
    const uint32_t on = mask4<VEC>(a.mask, r * a.ld_mask + c, left);
    get4<BF16, VEC>(p, a.logprobs, r * a.ld_logprobs + c, left);
    if (a.ref) get4<BF16, VEC>(ref, a.ref, r * a.ld_ref + c, left);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (on >> i & 1u) {
        sum = __fadd_rn(sum, __fsub_rn(p[i], ref[i]));
        count += 1.0f;
      }
  }
  return make_float2(warp_sum(sum), warp_sum(count));
}

__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

__device__ __forceinline__ void preference_finish(const Preference& q) {
  const advopt_preference_loss_args& a = q.a;
  __shared__ double red[32][1];
  const float2* units = static_cast<const float2*>(a.work);
  // a row's reward, in double, and its tokens (1 for a sum), behind the units' sums
  each_row<2>(2 * a.pairs, q.per_row, [&](double (&s)[2], int64_t u) {
    const float2 v = units[u];
    s[0] += v.x; s[1] += v.y;
  }, [&](int64_t r, const double (&s)[2]) {
    const double n = a.average && s[1] > 0.0 ? s[1] : 1.0;
    q.a.rewards[r] = (float)((double)a.beta * (s[0] / n));
    static_cast<double2*>(a.work)[q.per_row * a.pairs + r] = make_double2((double)a.beta * (s[0] / n), n);
  });
  __syncthreads();
  const double2* rows = static_cast<const double2*>(a.work) + q.per_row * a.pairs;
  double t[1] = {};
  for (int64_t i = threadIdx.x; i < a.pairs; i += FINISH) {
    const double2 c = rows[i], j = rows[i + a.pairs];
    const double h = c.x - j.x, e = a.smoothing;
    t[0] += (e < 1.0 ? (1.0 - e) * softplus(-h) : 0.0) + (e > 0.0 ? e * softplus(h) : 0.0);   // infinite without weight: nothing
    if (a.slope) {
      const double k = (double)a.beta / (double)a.pairs * (e - 1.0 / (1.0 + exp(h)));   // -(1 - e) sig(-h) + e sig(h)
      a.slope[i] = (float)(k / c.y);
      a.slope[i + a.pairs] = (float)(-k / j.y);
    }
  }
  cta_sum<1>(t, red);
  if (threadIdx.x == 0) *a.loss = (float)(t[0] / (double)a.pairs);
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void preference_units(const Preference& q, int64_t first, int64_t step) {
  for (int64_t u = first; u < 2 * q.a.pairs * q.per_row; u += step) {
    const int64_t r = u / q.per_row;
    const float2 v = preference_unit<BF16, VEC>(q, r, (u - r * q.per_row) * q.unit);
    if ((threadIdx.x & 31) == 0) static_cast<float2*>(q.a.work)[u] = v;
  }
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) preference_kernel(const __grid_constant__ Preference q) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  preference_units<BF16, VEC>(q, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), (int64_t)gridDim.x * 8);
}
__global__ void __launch_bounds__(FINISH) preference_finish_kernel(const __grid_constant__ Preference q) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  preference_finish(q);
}
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(FINISH) preference_one_kernel(const __grid_constant__ Preference q) {
  preference_units<BF16, VEC>(q, threadIdx.x >> 5, FINISH / 32);
  __syncthreads();
  preference_finish(q);
}

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) preference_grad_kernel(void* out, const float* dloss, const float* slope, const uint8_t* mask, int64_t ld_mask,
                                                              int64_t rows, int64_t cols, int64_t per_row) {
  const float d = *dloss;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * per_row; u += (int64_t)gridDim.x * 8) {
    const int64_t r = u / per_row, c0 = (u - r * per_row) * GRAD_UNIT, end = cols < c0 + GRAD_UNIT ? cols : c0 + GRAD_UNIT;
    const float k = __fmul_rn(d, slope[r]);
#pragma unroll
    for (int j = 0; j < GRAD_UNIT / BLOCK; ++j) {
      const int64_t c = c0 + j * BLOCK;
      const uint32_t on = mask4<VEC>(mask, r * ld_mask + c, end - c);
      const float v[4] = {on & 1u ? k : 0.0f, on & 2u ? k : 0.0f, on & 4u ? k : 0.0f, on & 8u ? k : 0.0f};
      put4<BF16, VEC>(out, r * cols + c, end - c, v);
    }
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
// Whether rows of elements of `size` bytes may be read four elements at a time; a row's last ones then are in the row's last whole four.
inline bool fours(const void* p, int64_t ld, int64_t rows, int size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && (rows <= 1 || ld % 4 == 0));
}

// `one` for few units; else `many`, and `finish` behind it, whose launch does not wait for its end.
template <class Q, class K>
cudaError_t run(const Q& q, int64_t units, K one, K many, K finish, cudaStream_t s) {
  if (units <= ONE_CTA) {
    one<<<1, FINISH, 0, s>>>(q);
    return cudaGetLastError();
  }
  many<<<grid_of(units), 256, 0, s>>>(q);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute behind;
  behind.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  behind.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(1);
  config.blockDim = dim3(FINISH);
  config.stream = s;
  config.attrs = &behind;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, finish, q);
}

}  // namespace loss
}  // namespace advopt

using namespace advopt;

extern "C" int64_t advopt_policy_loss_work(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : rows * ceil_div(cols, loss::unit_of(rows, cols)) * 16;
}

extern "C" int advopt_policy_loss(const advopt_policy_loss_args* a, void* stream) {
  if (!a || !loss::sizes_ok(a->rows, a->cols) || !a->loss || !a->kl || !a->clipped || !(a->clip_low >= 0.0f && a->clip_low <= 1.0f) ||
      !(a->clip_high >= 0.0f) || !(a->kl_weight - a->kl_weight == 0.0f))
    return set_error(ADVOPT_E_INVALID, "advopt_policy_loss: bad arguments");
  if (!known_dtype(a->dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_policy_loss: float32 and bfloat16 are supported");
  const bool any = a->rows && a->cols;
  if (any && (!a->scale || !a->logprobs || !a->old || !a->advantages || !a->work || !aligned16(a->work) ||
              !loss::pitch_ok(a->ld_logprobs, a->rows, a->cols) || !loss::pitch_ok(a->ld_old, a->rows, a->cols) ||
              (a->ref && !loss::pitch_ok(a->ld_ref, a->rows, a->cols)) || (a->mask && !loss::pitch_ok(a->ld_mask, a->rows, a->cols)) ||
              (a->ld_adv >= 0 && !loss::pitch_ok(a->ld_adv, a->rows, a->cols))))
    return set_error(ADVOPT_E_INVALID, "advopt_policy_loss: null or unaligned pointer, or a pitch below the row's length");
  loss::Policy q;
  q.a = *a;
  if (!any) q.a.rows = 0;
  q.unit = loss::unit_of(q.a.rows, a->cols);
  q.per_row = ceil_div(a->cols, q.unit);
  q.high32 = (float)a->log_high;
  q.low32 = (float)a->log_low;
  const int size = bytes_of(a->dtype);
  const bool vec = a->cols % 4 == 0 && loss::fours(a->logprobs, a->ld_logprobs, a->rows, size) && loss::fours(a->old, a->ld_old, a->rows, size) &&
                   loss::fours(a->ref, a->ld_ref, a->rows, size) && loss::fours(a->mask, a->ld_mask, a->rows, 1) &&
                   (a->ld_adv < 0 || loss::fours(a->advantages, a->ld_adv, a->rows, size)) && aligned16(a->slope);
  const int64_t units = q.a.rows * q.per_row;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  using namespace loss;
  const cudaError_t e = a->dtype == ADVOPT_DT_BF16
                            ? vec ? run(q, units, policy_one_kernel<true, true>, policy_kernel<true, true>, policy_finish_kernel, s)
                                  : run(q, units, policy_one_kernel<true, false>, policy_kernel<true, false>, policy_finish_kernel, s)
                            : vec ? run(q, units, policy_one_kernel<false, true>, policy_kernel<false, true>, policy_finish_kernel, s)
                                  : run(q, units, policy_one_kernel<false, false>, policy_kernel<false, false>, policy_finish_kernel, s);
  return check_cuda(e, "advopt_policy_loss");
}

extern "C" int advopt_policy_loss_grad(void* out, const float* dloss, const float* slope, const float* scale, int64_t rows, int64_t cols,
                                       int32_t dtype, void* stream) {
  if (!loss::sizes_ok(rows, cols)) return set_error(ADVOPT_E_INVALID, "advopt_policy_loss_grad: bad arguments");
  if (!known_dtype(dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_policy_loss_grad: float32 and bfloat16 are supported");
  if (rows == 0 || cols == 0) return ADVOPT_OK;
  if (!out || !dloss || !slope || !scale) return set_error(ADVOPT_E_INVALID, "advopt_policy_loss_grad: null pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t per_row = ceil_div(cols, loss::GRAD_UNIT);
  const unsigned grid = loss::grid_of(rows * per_row);
  const bool bf16 = dtype == ADVOPT_DT_BF16, vec = cols % 4 == 0 && aligned16(out) && aligned16(slope);
  if (bf16 && vec) loss::policy_grad_kernel<true, true><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  else if (bf16) loss::policy_grad_kernel<true, false><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  else if (vec) loss::policy_grad_kernel<false, true><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  else loss::policy_grad_kernel<false, false><<<grid, 256, 0, s>>>(out, dloss, slope, scale, rows, cols, per_row);
  return check_cuda(cudaGetLastError(), "advopt_policy_loss_grad");
}

extern "C" int64_t advopt_preference_loss_work(int64_t pairs, int64_t cols) {
  if (pairs <= 0) return 0;
  const int64_t rows = 2 * pairs;
  // the units' sums, then a row's reward and tokens
  return rows * ceil_div(cols > 0 ? cols : 0, loss::unit_of(rows, cols)) * 8 + rows * 16;
}

extern "C" int advopt_preference_loss(const advopt_preference_loss_args* a, void* stream) {
  if (!a || a->pairs < 1 || a->pairs >= (int64_t)1 << 30 || !loss::sizes_ok(2 * a->pairs, a->cols) || !a->loss || !a->rewards ||
      !(a->beta - a->beta == 0.0f) || !(a->smoothing >= 0.0f && a->smoothing <= 1.0f))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss: bad arguments");
  if (!known_dtype(a->dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_preference_loss: float32 and bfloat16 are supported");
  const int64_t rows = 2 * a->pairs;
  if (!a->work || !aligned16(a->work) || (a->cols && (!a->logprobs || !loss::pitch_ok(a->ld_logprobs, rows, a->cols) ||
                  (a->ref && !loss::pitch_ok(a->ld_ref, rows, a->cols)) || (a->mask && !loss::pitch_ok(a->ld_mask, rows, a->cols)))))
    return set_error(ADVOPT_E_INVALID, "advopt_preference_loss: null or unaligned pointer, or a pitch below the row's length");
  loss::Preference q;
  q.a = *a;
  q.unit = loss::unit_of(rows, a->cols);
  q.per_row = ceil_div(a->cols, q.unit);
  const int size = bytes_of(a->dtype);
  const bool vec = a->cols % 4 == 0 && loss::fours(a->logprobs, a->ld_logprobs, rows, size) && loss::fours(a->ref, a->ld_ref, rows, size) &&
                   loss::fours(a->mask, a->ld_mask, rows, 1);
  const int64_t units = rows * q.per_row;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  using namespace loss;
  const cudaError_t e =
      a->dtype == ADVOPT_DT_BF16
          ? vec ? run(q, units, preference_one_kernel<true, true>, preference_kernel<true, true>, preference_finish_kernel, s)
                : run(q, units, preference_one_kernel<true, false>, preference_kernel<true, false>, preference_finish_kernel, s)
          : vec ? run(q, units, preference_one_kernel<false, true>, preference_kernel<false, true>, preference_finish_kernel, s)
                : run(q, units, preference_one_kernel<false, false>, preference_kernel<false, false>, preference_finish_kernel, s);
  return check_cuda(e, "advopt_preference_loss");
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
  const int64_t rows = 2 * pairs, per_row = ceil_div(cols, loss::GRAD_UNIT);
  const unsigned grid = loss::grid_of(rows * per_row);
  const bool bf16 = dtype == ADVOPT_DT_BF16, vec = cols % 4 == 0 && aligned16(out) && loss::fours(mask, ld_mask, rows, 1);
  if (bf16 && vec) loss::preference_grad_kernel<true, true><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, rows, cols, per_row);
  else if (bf16) loss::preference_grad_kernel<true, false><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, rows, cols, per_row);
  else if (vec) loss::preference_grad_kernel<false, true><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, rows, cols, per_row);
  else loss::preference_grad_kernel<false, false><<<grid, 256, 0, s>>>(out, dloss, slope, mask, ld_mask, rows, cols, per_row);
  return check_cuda(cudaGetLastError(), "advopt_preference_loss_grad");
}
