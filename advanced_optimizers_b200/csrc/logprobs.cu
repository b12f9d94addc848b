// Log-probabilities of given tokens: lp_r = z_k - log sum_j e^(z_j) with z the
// row of logits over the temperature, and dlogits = dlp / temperature *
// ((j == k) - p_j).
//
// Forward: one pass with a running maximum m and sum s of e^(z - m), rescaled
// when the maximum grows; threads, warps and the CTAs of a cluster are joined
// the same way.  The pair (m, s) is kept, so that the backward pass has p_j =
// e^(z_j - m) / s without the rounding of m + log s.  Backward: elementwise.
// Both are bound by HBM; an exponential an element is the next limit (16 a
// clock and SM, 4.6e12 a second; bf16 logits arrive at 3.3e12).
#include <cooperative_groups.h>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace advopt {
namespace lp {

namespace cg = cooperative_groups;

constexpr float NEG_INF = -__builtin_huge_valf();

// 2^x for x <= 0 (off by at most 2^-22 of it); results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Args {
  float* out;
  float* stats;
  const void* logits;
  const void* tokens;
  int32_t* err;
  int64_t inner, ld_outer, ld_inner, rows;
  int64_t ignore;
  uint32_t vocab;
  int wide;
  float c;                  // log2(e) / temperature
  float inv;                // 1 / temperature
};

__device__ __forceinline__ int64_t row_start(const Args& a, int64_t r) {
  const int64_t o = a.inner >= a.rows ? 0 : r / a.inner;
  return o * a.ld_outer + (r - o * a.inner) * a.ld_inner;
}
__device__ __forceinline__ int64_t token_of(const Args& a, int64_t r) {
  return a.wide ? static_cast<const int64_t*>(a.tokens)[r] : (int64_t) static_cast<const int32_t*>(a.tokens)[r];
}

// A running maximum and sum of 2^((x - m) c).  NaN does not enter the maximum
// but the sum, and so does an infinity (inf - inf).
struct Run {
  float m = NEG_INF, s = 0.0f;
  __device__ __forceinline__ static float base(float m) { return m == NEG_INF ? 0.0f : m; }
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > m) {
      s = __fmul_rn(s, exp2_fast(__fmul_rn(__fsub_rn(m, top), c)));
      m = top;
    }
  }
  __device__ __forceinline__ void join(float om, float os, float c) {
    const float top = fmaxf(m, om), b = base(top);
    s = __fadd_rn(__fmul_rn(s, exp2_fast(__fmul_rn(__fsub_rn(m, b), c))), __fmul_rn(os, exp2_fast(__fmul_rn(__fsub_rn(om, b), c))));
    m = top;
  }
  __device__ __forceinline__ void add(float x, float c) {
    raise(x, c);
    s = __fadd_rn(s, exp2_fast(__fmul_rn(__fsub_rn(x, base(m)), c)));
  }
};

// 16 bytes of logits.
template <bool BF16>
struct Vec {
  static constexpr int E = BF16 ? 8 : 4;
  uint4 q;
  __device__ __forceinline__ float at(int e) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    return BF16 ? u2f((e & 1) ? w[(e >> 1) & 3] & 0xFFFF0000u : w[(e >> 1) & 3] << 16) : u2f(w[e & 3]);
  }
};
template <bool BF16>
__device__ __forceinline__ float one(const void* base, int64_t k) {
  return BF16 ? bf16_to_f(__ldg(static_cast<const uint16_t*>(base) + k)) : __ldg(static_cast<const float*>(base) + k);
}

// Elements ahead of the first 16-byte boundary.
template <bool BF16>
__device__ __forceinline__ uint32_t head_of(const void* p, uint32_t n) {
  const uint32_t h = (uint32_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (BF16 ? 2 : 4);
  return h < n ? h : n;
}

constexpr int U = 4;   // 16-byte loads that a thread has on their way

// The part `rank` of `ranks` of a row, by `width` threads.
template <bool BF16>
__device__ __forceinline__ void scan(Run& run, const void* row, uint32_t n, float c, int thread, int width, uint32_t rank, uint32_t ranks) {
  constexpr int E = Vec<BF16>::E;
  const uint32_t head = head_of<BF16>(row, n), vecs = (n - head) / E, tail = head + vecs * E;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(row) + head * (BF16 ? 2 : 4));
  uint32_t i = (uint32_t)((uint64_t)vecs * rank / ranks) + thread;
  const uint32_t end = (uint32_t)((uint64_t)vecs * (rank + 1) / ranks);
  for (; i < end; i += U * width) {
    Vec<BF16> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u].q = i + u * width < end ? __ldg(p + i + u * width)
                                   : (BF16 ? make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u)
                                           : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u));   // -infinity
    float top = NEG_INF;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) top = fmaxf(top, v[u].at(e));
    run.raise(top, c);
    const float b = -Run::base(run.m);
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 d = mul2(add2(make_float2(v[u].at(e), v[u].at(e + 1)), splat2(b)), splat2(c));
        s = add2(s, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
      }
    run.s = __fadd_rn(run.s, __fadd_rn(s.x, s.y));
  }
  if (rank == 0) {
    for (uint32_t k = thread; k < head; k += width) run.add(one<BF16>(row, k), c);
    for (uint32_t k = tail + thread; k < n; k += width) run.add(one<BF16>(row, k), c);
  }
}

__device__ __forceinline__ void warp_join(Run& run, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) run.join(__shfl_xor_sync(0xffffffffu, run.m, o), __shfl_xor_sync(0xffffffffu, run.s, o), c);
}

template <bool BF16>
__device__ __forceinline__ void finish(const Args& a, int64_t r, const void* row, int64_t token, const Run& run) {
  float v = u2f(0x7fc00000u);
  if (token >= 0 && token < (int64_t)a.vocab)
    v = __fsub_rn(__fmul_rn(__fsub_rn(one<BF16>(row, token), run.m), a.inv), logf(run.s));
  else if (a.err)
    *reinterpret_cast<volatile int32_t*>(a.err) = 1;
  a.out[r] = v;
  if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(run.m, run.s);
}

template <bool BF16>
__device__ __forceinline__ const void* row_of(const Args& a, int64_t r) {
  return static_cast<const unsigned char*>(a.logits) + row_start(a, r) * (BF16 ? 2 : 4);
}

constexpr int THREADS = 512;

// A cluster of CL CTAs per row.
template <bool BF16, int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(THREADS) forward_kernel(const __grid_constant__ Args a) {
  __shared__ float2 red[2][THREADS / 32];
  __shared__ float2 whole[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = blockIdx.x % CL;
  int round = 0;
  for (int64_t r = blockIdx.x / CL; r < a.rows; r += gridDim.x / CL) {
    const int64_t token = token_of(a, r);
    if (token == a.ignore) {
      if (rank == 0 && threadIdx.x == 0) {
        a.out[r] = 0.0f;
        if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(0.0f, 1.0f);
      }
      continue;
    }
    const void* row = row_of<BF16>(a, r);
    Run run;
    scan<BF16>(run, row, a.vocab, a.c, threadIdx.x, THREADS, rank, CL);
    warp_join(run, a.c);
    if (lane == 0) red[round][warp] = make_float2(run.m, run.s);
    __syncthreads();
    if (warp == 0) {
      const float2 t = lane < THREADS / 32 ? red[round][lane] : make_float2(NEG_INF, 0.0f);
      run.m = t.x;
      run.s = t.y;
      warp_join(run, a.c);
    }
    if (CL > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (threadIdx.x == 0) whole[round] = make_float2(run.m, run.s);
      cluster.sync();
      if (rank == 0 && threadIdx.x == 0) {
#pragma unroll
        for (int k = 1; k < CL; ++k) {
          const float2 t = *cluster.map_shared_rank(&whole[round], k);
          run.join(t.x, t.y, a.c);
        }
      }
    }
    if (rank == 0 && threadIdx.x == 0) finish<BF16>(a, r, row, token, run);
    round ^= 1;
  }
  if (CL > 1) cg::this_cluster().sync();   // no CTA ends while its sums are read
}

// A warp per row.
template <bool BF16>
__global__ void __launch_bounds__(256) short_forward_kernel(const __grid_constant__ Args a) {
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows; r += (int64_t)gridDim.x * 8) {
    const int64_t token = token_of(a, r);
    if (token == a.ignore) {
      if (lane == 0) {
        a.out[r] = 0.0f;
        if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(0.0f, 1.0f);
      }
      continue;
    }
    const void* row = row_of<BF16>(a, r);
    Run run;
    scan<BF16>(run, row, a.vocab, a.c, lane, 32, 0, 1);
    warp_join(run, a.c);
    if (lane == 0) finish<BF16>(a, r, row, token, run);
  }
}

// ---- backward: a CTA per row and 256 * U times 16 bytes of dlogits ----
constexpr int GRAD_THREADS = 256;

template <bool BF16>
__global__ void __launch_bounds__(GRAD_THREADS) grad_kernel(void* dlogits, const float* dlp, const __grid_constant__ Args a, uint32_t segs) {
  constexpr int E = Vec<BF16>::E;
  const int64_t units = a.rows * segs;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t r = units >> 32 ? unit / segs : (int64_t)((uint32_t)unit / segs);
    const uint32_t seg = (uint32_t)(unit - r * segs);
    const float g = __ldg(dlp + r);
    const int64_t token = token_of(a, r);
    const bool zero = g == 0.0f || token == a.ignore;
    const bool bad = !zero && (token < 0 || token >= (int64_t)a.vocab);
    unsigned char* out = static_cast<unsigned char*>(dlogits) + r * a.vocab * (BF16 ? 2 : 4);
    const unsigned char* in = static_cast<const unsigned char*>(row_of<BF16>(a, r));
    const uint32_t n = a.vocab, head = head_of<BF16>(out, n), vecs = (n - head) / E, tail = head + vecs * E;
    const float2 st = zero ? make_float2(0.0f, 1.0f) : __ldg(reinterpret_cast<const float2*>(a.stats + 2 * r));
    const float at_token = bad ? u2f(0x7fc00000u) : __fmul_rn(g, a.inv);   // a row without a token is NaN
    const float k = -__fdiv_rn(at_token, st.y), m = st.x;
    const uint32_t target = zero ? 0xffffffffu : (uint32_t)token;
    const auto value = [&](float x, uint32_t j) {
      const float v = __fmul_rn(k, exp2_fast(__fmul_rn(__fsub_rn(x, m), a.c)));
      return j == target ? __fadd_rn(v, at_token) : v;
    };
    const auto put = [&](uint32_t j) {
      const float v = zero ? 0.0f : value(one<BF16>(in, j), j);
      if (BF16) reinterpret_cast<uint16_t*>(out)[j] = (uint16_t)f_to_bf16_rne(v);
      else reinterpret_cast<float*>(out)[j] = v;
    };
    if (seg == 0) {
      for (uint32_t j = threadIdx.x; j < head; j += GRAD_THREADS) put(j);
      for (uint32_t j = tail + threadIdx.x; j < n; j += GRAD_THREADS) put(j);
    }
    uint4* to = reinterpret_cast<uint4*>(out + head * (BF16 ? 2 : 4));
    const uint32_t i0 = seg * (GRAD_THREADS * U) + threadIdx.x;
    if (zero) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * GRAD_THREADS < vecs) to[i0 + u * GRAD_THREADS] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const unsigned char* body = in + head * (BF16 ? 2 : 4);
    const bool whole = (reinterpret_cast<uintptr_t>(body) & 15) == 0;
    Vec<BF16> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * GRAD_THREADS;
      if (i >= vecs) continue;
      if (whole) {
        v[u].q = __ldg(reinterpret_cast<const uint4*>(body) + i);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (BF16) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(body) + i * 8 + 2 * e;
            w[e] = (uint32_t)__ldg(p) | (uint32_t)__ldg(p + 1) << 16;
          } else {
            w[e] = __ldg(reinterpret_cast<const uint32_t*>(body) + i * 4 + e);
          }
        }
        v[u].q = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * GRAD_THREADS;
      if (i >= vecs) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 d = mul2(add2(make_float2(v[u].at(e), v[u].at(e + 1)), splat2(-m)), splat2(a.c));
        const float2 p = mul2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), splat2(k));
        o[e] = p.x;
        o[e + 1] = p.y;
      }
      const uint32_t behind = target - (head + i * E);
      if (behind < (uint32_t)E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((int)behind == e) o[e] = __fadd_rn(o[e], at_token);
      }
      if constexpr (BF16) to[i] = make_uint4(bf16x2(o[0], o[1]), bf16x2(o[2], o[3]), bf16x2(o[4], o[5]), bf16x2(o[6], o[7]));
      else to[i] = make_uint4(f2u(o[0]), f2u(o[1]), f2u(o[2]), f2u(o[3]));
    }
  }
}

constexpr int64_t SMS = 148;

template <bool BF16, int CL>
void launch(const Args& a, cudaStream_t s) {
  const int64_t most = SMS * 4 / CL;
  forward_kernel<BF16, CL><<<(unsigned)((a.rows < most ? a.rows : most) * CL), THREADS, 0, s>>>(a);
}

template <bool BF16>
void forward(const Args& a, cudaStream_t s) {
  const int64_t bytes = (int64_t)a.vocab * (BF16 ? 2 : 4);
  if (bytes <= 8192) {
    const int64_t ctas = ceil_div(a.rows, 8);
    short_forward_kernel<BF16><<<(unsigned)(ctas < SMS * 8 ? ctas : SMS * 8), 256, 0, s>>>(a);
    return;
  }
  // a row is split while that gives the SMs more than one CTA each and a CTA at least 32 KB
  int cl = 1;
  while (cl < 8 && a.rows * cl < 2 * SMS && bytes >= cl * 65536) cl *= 2;
  if (cl == 8) launch<BF16, 8>(a, s);
  else if (cl == 4) launch<BF16, 4>(a, s);
  else if (cl == 2) launch<BF16, 2>(a, s);
  else launch<BF16, 1>(a, s);
}

// nullptr when the arguments are fine.
const char* check(const advopt_token_logprobs_args* a) {
  if (!a || a->rows < 0 || a->rows >= (int64_t)1 << 40 || a->vocab < 1 || a->vocab >= (int64_t)1 << 31 || a->inner < 1 ||
      (a->token_bytes != 4 && a->token_bytes != 8) || !(a->temperature > 0.0f) || a->temperature > 3e38f)
    return "token_logprobs: bad arguments";
  if (!known_dtype(a->dtype)) return "token_logprobs: float32 and bfloat16 logits are supported";
  if (a->rows && (!a->logits || !a->tokens || reinterpret_cast<uintptr_t>(a->stats) % 8)) return "token_logprobs: null or unaligned pointer";
  return nullptr;
}
Args args_of(const advopt_token_logprobs_args& a) {
  const double inv = 1.0 / (double)a.temperature;
  return {a.logprobs, a.stats, a.logits, a.tokens, a.err, a.inner, a.ld_outer, a.ld_inner, a.rows, a.ignore, (uint32_t)a.vocab,
          a.token_bytes == 8, (float)(inv * 1.4426950408889634), (float)inv};
}

}  // namespace lp
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_token_logprobs(const advopt_token_logprobs_args* a, void* stream) {
  if (const char* why = lp::check(a)) return set_error(ADVOPT_E_INVALID, why);
  if (a->rows == 0) return ADVOPT_OK;
  if (!a->logprobs) return set_error(ADVOPT_E_INVALID, "token_logprobs: null output");
  if (a->dtype == ADVOPT_DT_BF16) lp::forward<true>(lp::args_of(*a), static_cast<cudaStream_t>(stream));
  else lp::forward<false>(lp::args_of(*a), static_cast<cudaStream_t>(stream));
  return check_cuda(cudaGetLastError(), "advopt_token_logprobs");
}

extern "C" int advopt_token_logprobs_grad(void* dlogits, const float* dlogprobs, const advopt_token_logprobs_args* a, void* stream) {
  if (const char* why = lp::check(a)) return set_error(ADVOPT_E_INVALID, why);
  if (a->rows == 0) return ADVOPT_OK;
  if (!dlogits || !dlogprobs || !a->stats) return set_error(ADVOPT_E_INVALID, "token_logprobs_grad: null pointer");
  const bool bf16 = a->dtype == ADVOPT_DT_BF16;
  const int64_t segs = ceil_div(a->vocab, lp::GRAD_THREADS * lp::U * (bf16 ? 8 : 4)), units = a->rows * segs;
  const unsigned grid = (unsigned)(units < 0x7fffffff ? units : 0x7fffffff);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (bf16) lp::grad_kernel<true><<<grid, lp::GRAD_THREADS, 0, s>>>(dlogits, dlogprobs, lp::args_of(*a), (uint32_t)segs);
  else lp::grad_kernel<false><<<grid, lp::GRAD_THREADS, 0, s>>>(dlogits, dlogprobs, lp::args_of(*a), (uint32_t)segs);
  return check_cuda(cudaGetLastError(), "advopt_token_logprobs_grad");
}
