// Log-probabilities of given tokens: lp_r = z_k - log sum_j e^(z_j) with z the
// row of logits over the temperature, and dlogits = dlp / temperature *
// ((j == k) - p_j).
//
// Forward: one pass with a running maximum m and sum s of e^(z - m), rescaled
// when the maximum grows; threads, warps and parts of a row are joined the same
// way.  The pair (m, 1 / s) is kept, so that the backward pass has p_j =
// e^(z_j - m) / s without the rounding of m + log s.  Backward: elementwise.
// Both are bound by HBM; an exponential an element is the next limit (16 a
// clock and SM, 4.6e12 a second; bf16 logits arrive at 3.3e12).
//
// The lanes of a warp take 6 KB of a row at once (backward 4), all of it on its
// way before the first element is looked at, and the warp ends: no loop, no
// barrier, and the warps behind it keep HBM busy meanwhile (a read with an exponential and
// a maximum an element: 144 us for 4096 x 128256 bf16; with a CTA that walks
// along a row, however its loads were scheduled, 172 to 201).  Parts of longer
// rows are joined by a second launch; rows up to 1 KB share a warp.
#include <cooperative_groups.h>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace advopt {
namespace lp {

constexpr float NEG_INF = -__builtin_huge_valf();

// 2^x for x <= 0 (off by at most 2^-22 of it); results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct Args {
  float* out;
  float* stats;             // {m, 1 / s}
  float2* part;             // {m, s} of the parts of rows, [rows][parts]
  const void* logits;
  const void* tokens;
  int32_t* err;
  int64_t inner, ld_outer, ld_inner, rows;
  int64_t ignore;
  uint32_t vocab, parts;
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

// The largest element, NaN left out; bf16 ones two at a time.
template <bool BF16, int U>
__device__ __forceinline__ float largest(const Vec<BF16> (&v)[U]) {
  if constexpr (BF16) {
    uint32_t m = 0xFF80FF80u;
#pragma unroll
    for (int u = 0; u < U; ++u) m = max_bf16x2(max_bf16x2(max_bf16x2(v[u].q.x, v[u].q.y), max_bf16x2(v[u].q.z, v[u].q.w)), m);
    return fmaxf(u2f(m << 16), u2f(m & 0xFFFF0000u));
  } else {
    float m = NEG_INF;
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(fmaxf(fmaxf(v[u].at(0), v[u].at(1)), fmaxf(v[u].at(2), v[u].at(3))), m);
    return m;
  }
}

constexpr int THREADS = 256;

// L lanes take U vectors of 16 bytes each of a row at once: 512 bytes, 1 KB, or
// 6 KB (backward 4), which are a part of a longer row.
template <int L, bool BACK>
struct Share {
  static constexpr int U = L == 32 ? (BACK ? 8 : 12) : 4, VECS = L * U;
};

// Their running maximum and sum of part `part` of a row; the first part's
// lanes also take what lies ahead of the row's first 16-byte boundary and
// behind its last one.
template <bool BF16, int L>
__device__ __forceinline__ void scan(Run& run, const void* row, uint32_t n, float c, int lane, uint32_t part) {
  constexpr int E = Vec<BF16>::E, U = Share<L, false>::U;
  const uint32_t head = head_of<BF16>(row, n), vecs = (n - head) / E, tail = head + vecs * E;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(row) + head * (BF16 ? 2 : 4));
  const uint32_t i = part * Share<L, false>::VECS + lane;
  Vec<BF16> v[U];
  p += i;
  if (part * Share<L, false>::VECS + Share<L, false>::VECS <= vecs) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].q = __ldg(p + u * L);
  } else {
    const uint4 nothing = BF16 ? make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u)
                               : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);   // -infinity
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].q = i + u * L < vecs ? __ldg(p + u * L) : nothing;
  }
  const float top = largest<BF16, U>(v);
  run.m = top;
  const float2 b = splat2(-Run::base(top));
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 d = mul2(add2(make_float2(v[u].at(e), v[u].at(e + 1)), b), splat2(c));
      s = add2(s, make_float2(exp2_fast(d.x), exp2_fast(d.y)));
    }
  run.s = __fadd_rn(s.x, s.y);
  if (part == 0) {
    for (uint32_t k = lane; k < head; k += L) run.add(one<BF16>(row, k), c);
    for (uint32_t k = tail + lane; k < n; k += L) run.add(one<BF16>(row, k), c);
  }
}

// The sums of the L lanes of a group, in all of them: the largest maximum first,
// so that each lane rescales once.
template <int L>
__device__ __forceinline__ void join_lanes(Run& run, float c) {
  float top = run.m;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // m - top of two infinities: nothing was added below it, or the sum is NaN already
  run.s = __fmul_rn(run.s, exp2_fast(__fmul_rn(__fsub_rn(run.m, Run::base(top)), c)));
  run.m = top;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) run.s = __fadd_rn(run.s, __shfl_xor_sync(0xffffffffu, run.s, o));
}

template <bool BF16>
__device__ __forceinline__ const void* row_of(const Args& a, int64_t r) {
  return static_cast<const unsigned char*>(a.logits) + row_start(a, r) * (BF16 ? 2 : 4);
}

template <bool BF16>
__device__ __forceinline__ void finish(const Args& a, int64_t r, int64_t token, const Run& run) {
  float v = u2f(0x7fc00000u);
  if (token >= 0 && token < (int64_t)a.vocab)
    v = __fsub_rn(__fmul_rn(__fsub_rn(one<BF16>(row_of<BF16>(a, r), token), run.m), a.inv), logf(run.s));
  else if (a.err)
    *reinterpret_cast<volatile int32_t*>(a.err) = 1;
  a.out[r] = v;
  if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(run.m, __fdiv_rn(1.0f, run.s));
}
__device__ __forceinline__ void ignored(const Args& a, int64_t r) {
  a.out[r] = 0.0f;
  if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(0.0f, 0.0f);
}

// Row and part of a group of lanes; rows behind the last one: a.rows.
struct Place {
  int64_t r;
  uint32_t part;
  template <int L>
  __device__ __forceinline__ static Place of(const Args& a) {
    const int64_t u = (int64_t)blockIdx.x * (THREADS / L) + threadIdx.x / L;
    if (L < 32 || a.parts == 1) return {u < a.rows ? u : a.rows, 0};
    const int64_t r = u >> 32 ? u / a.parts : (int64_t)((uint32_t)u / a.parts);
    return {r < a.rows ? r : a.rows, (uint32_t)(u - r * a.parts)};
  }
};

template <bool BF16, int L>
__global__ void __launch_bounds__(THREADS, 4) forward_kernel(const __grid_constant__ Args a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & (L - 1);
  const Place at = Place::of<L>(a);
  const bool there = at.r < a.rows;
  const int64_t token = there ? token_of(a, at.r) : a.ignore;
  Run run;
  if (token != a.ignore) scan<BF16, L>(run, row_of<BF16>(a, at.r), a.vocab, a.c, lane, at.part);
  join_lanes<L>(run, a.c);   // all groups of the warp take part
  if (lane || !there) return;
  if (L == 32 && a.parts > 1) a.part[at.r * a.parts + at.part] = make_float2(run.m, run.s);
  else if (token == a.ignore) ignored(a, at.r);
  else finish<BF16>(a, at.r, token, run);
}

// A cluster per row, for as many rows as there are SMs: they are bound by
// latency, which a second launch and its buffer would add to.
constexpr int CLUSTER = 8, WARPS = THREADS / 32;

template <bool BF16>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS) row_kernel(const __grid_constant__ Args a) {
  namespace cg = cooperative_groups;
  __shared__ float2 red[WARPS], whole;
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster.block_rank();
  const int64_t r = blockIdx.x / CLUSTER, token = token_of(a, r);
  if (token == a.ignore) {   // of all the cluster's CTAs
    if (rank == 0 && threadIdx.x == 0) ignored(a, r);
    return;
  }
  Run run;
  for (uint32_t part = rank * WARPS + warp; part < a.parts; part += CLUSTER * WARPS) {
    Run more;
    scan<BF16, 32>(more, row_of<BF16>(a, r), a.vocab, a.c, lane, part);
    run.join(more.m, more.s, a.c);
  }
  join_lanes<32>(run, a.c);
  if (lane == 0) red[warp] = make_float2(run.m, run.s);
  __syncthreads();
  if (warp == 0) {
    run.m = red[lane & (WARPS - 1)].x;
    run.s = red[lane & (WARPS - 1)].y;
    join_lanes<WARPS>(run, a.c);
    if (lane == 0) whole = make_float2(run.m, run.s);
  }
  cluster.sync();
  if (rank == 0 && warp == 0) {
    const float2 t = *cluster.map_shared_rank(&whole, lane & (CLUSTER - 1));
    run.m = t.x;
    run.s = t.y;
    join_lanes<CLUSTER>(run, a.c);
    if (lane == 0) finish<BF16>(a, r, token, run);
  }
  cluster.sync();   // no CTA ends while its sums are read
}

// L lanes per row join its parts.
template <bool BF16, int L>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & (L - 1);
  const int64_t r = (int64_t)blockIdx.x * (THREADS / L) + threadIdx.x / L;
  const bool there = r < a.rows;
  const int64_t token = there ? token_of(a, r) : a.ignore;
  Run run;
  if (token != a.ignore)
    for (uint32_t k = lane; k < a.parts; k += L) {
      const float2 t = a.part[r * a.parts + k];
      run.join(t.x, t.y, a.c);
    }
  join_lanes<L>(run, a.c);
  if (lane || !there) return;
  if (token == a.ignore) ignored(a, r);
  else finish<BF16>(a, r, token, run);
}

// ---- backward: the same shares of dlogits ----
// Stores are of aligned 16 bytes of dlogits; the logits that belong to them are
// aligned too where they lie the same way, and else are read by aligned 16
// bytes, each of which holds one of them, and shifted.
template <bool BF16>
__device__ __forceinline__ uint4 shifted_load(const unsigned char* p) {
  const uint32_t o = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const uint4* base = reinterpret_cast<const uint4*>(p - o);
  const uint4 q = __ldg(base);
  if (o == 0) return q;
  const uint4 n = __ldg(base + 1);
  const bool by8 = o & 8, by4 = o & 4, by2 = o & 2;
  const uint32_t s[6] = {by8 ? q.z : q.x, by8 ? q.w : q.y, by8 ? n.x : q.z, by8 ? n.y : q.w, by8 ? n.z : n.x, by8 ? n.w : n.y};
  uint32_t t[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) t[i] = by4 ? s[i + 1] : s[i];
  if (BF16 && by2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __funnelshift_r(t[i], t[i + 1], 16);
  }
  return make_uint4(t[0], t[1], t[2], t[3]);
}

template <bool BF16, int L>
__global__ void __launch_bounds__(THREADS) grad_kernel(void* dlogits, const float* dlp, const __grid_constant__ Args a) {
  constexpr int E = Vec<BF16>::E, SIZE = BF16 ? 2 : 4, U = Share<L, true>::U;
  const int lane = threadIdx.x & (L - 1);
  const Place at = Place::of<L>(a);
  if (at.r >= a.rows) return;
  const float g = __ldg(dlp + at.r);
  const int64_t token = token_of(a, at.r);
  const float2 st = __ldg(reinterpret_cast<const float2*>(a.stats) + at.r);
  const bool zero = g == 0.0f || token == a.ignore;
  unsigned char* out = static_cast<unsigned char*>(dlogits) + at.r * a.vocab * SIZE;
  const uint32_t n = a.vocab, head = head_of<BF16>(out, n), vecs = (n - head) / E, tail = head + vecs * E;
  const uint32_t i0 = at.part * Share<L, true>::VECS + lane;
  uint4* to = reinterpret_cast<uint4*>(out + head * SIZE);
  const unsigned char* in = static_cast<const unsigned char*>(row_of<BF16>(a, at.r));
  if (zero) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * L < vecs) to[i0 + u * L] = make_uint4(0, 0, 0, 0);
  } else {
    Vec<BF16> v[U];
    if ((reinterpret_cast<uintptr_t>(in + head * SIZE) & 15) == 0) {
      const uint4* p = reinterpret_cast<const uint4*>(in + head * SIZE);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * L < vecs) v[u].q = __ldg(p + i0 + u * L);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * L < vecs) v[u].q = shifted_load<BF16>(in + (head + (i0 + u * L) * E) * (int64_t)SIZE);
    }
    // k e^((x - m) / temperature), and hit more at the token; a row without a token is NaN
    const float hit = token < 0 || token >= (int64_t)n ? u2f(0x7fc00000u) : __fmul_rn(g, a.inv);
    const float k = -__fmul_rn(hit, st.y);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * L;
      if (i >= vecs) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 d = mul2(add2(make_float2(v[u].at(e), v[u].at(e + 1)), splat2(-st.x)), splat2(a.c));
        const float2 q = mul2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), splat2(k));
        o[e] = q.x;
        o[e + 1] = q.y;
      }
      const uint32_t behind = (uint32_t)token - (head + i * E);
      if (behind < (uint32_t)E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((int)behind == e) o[e] = __fadd_rn(o[e], hit);
      }
      if constexpr (BF16) to[i] = make_uint4(bf16x2(o[0], o[1]), bf16x2(o[2], o[3]), bf16x2(o[4], o[5]), bf16x2(o[6], o[7]));
      else to[i] = make_uint4(f2u(o[0]), f2u(o[1]), f2u(o[2]), f2u(o[3]));
    }
    if (at.part == 0) {
      // fewer than E elements ahead of the first boundary, and behind the last
#pragma unroll
      for (int q = lane; q < 2 * E; q += L) {
        const uint32_t j = q < E ? q : tail + q - E;
        if (q < E ? j < head : j < n) {
          float x = __fmul_rn(k, exp2_fast(__fmul_rn(__fsub_rn(one<BF16>(in, j), st.x), a.c)));
          if (j == (uint32_t)token) x = __fadd_rn(x, hit);
          if (BF16) reinterpret_cast<uint16_t*>(out)[j] = (uint16_t)f_to_bf16_rne(x);
          else reinterpret_cast<float*>(out)[j] = x;
        }
      }
    }
    return;
  }
  if (at.part == 0) {
    for (uint32_t j = lane; j < head; j += L) {
      if (BF16) reinterpret_cast<uint16_t*>(out)[j] = 0;
      else reinterpret_cast<float*>(out)[j] = 0.0f;
    }
    for (uint32_t j = tail + lane; j < n; j += L) {
      if (BF16) reinterpret_cast<uint16_t*>(out)[j] = 0;
      else reinterpret_cast<float*>(out)[j] = 0.0f;
    }
  }
}

// Parts of a row, 1 where a group of lanes has all of it.
template <bool BACK>
inline int64_t parts_of(int64_t bytes) { return ceil_div(bytes, Share<32, BACK>::VECS * 16); }

// Whether each row is one cluster's.
inline bool alone(int64_t rows, int64_t parts) { return parts > 1 && rows <= 148; }

template <class K, class... A>
cudaError_t launch(K kernel, int lanes, int64_t groups, bool behind, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)ceil_div(groups, THREADS / lanes));
  config.blockDim = dim3(THREADS);
  config.stream = s;
  config.attrs = &at;
  config.numAttrs = behind ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <bool BF16>
cudaError_t forward(const Args& a, cudaStream_t s) {
  const int64_t bytes = (int64_t)a.vocab * (BF16 ? 2 : 4);
  if (bytes <= Share<8, false>::VECS * 16) return launch(forward_kernel<BF16, 8>, 8, a.rows, false, s, a);
  if (bytes <= Share<16, false>::VECS * 16) return launch(forward_kernel<BF16, 16>, 16, a.rows, false, s, a);
  if (alone(a.rows, a.parts)) {
    row_kernel<BF16><<<(unsigned)(a.rows * CLUSTER), THREADS, 0, s>>>(a);
    return cudaGetLastError();
  }
  const cudaError_t e = launch(forward_kernel<BF16, 32>, 32, a.rows * a.parts, false, s, a);
  if (e != cudaSuccess || a.parts == 1) return e;
  return a.parts <= 16 ? launch(join_kernel<BF16, 8>, 8, a.rows, true, s, a) : launch(join_kernel<BF16, 32>, 32, a.rows, true, s, a);
}

template <bool BF16>
cudaError_t grad(void* dlogits, const float* dlp, const Args& a, cudaStream_t s) {
  const int64_t bytes = (int64_t)a.vocab * (BF16 ? 2 : 4);
  if (bytes <= Share<8, true>::VECS * 16) return launch(grad_kernel<BF16, 8>, 8, a.rows, false, s, dlogits, dlp, a);
  if (bytes <= Share<16, true>::VECS * 16) return launch(grad_kernel<BF16, 16>, 16, a.rows, false, s, dlogits, dlp, a);
  return launch(grad_kernel<BF16, 32>, 32, a.rows * a.parts, false, s, dlogits, dlp, a);
}

// nullptr when the arguments are fine.
const char* check(const advopt_token_logprobs_args* a) {
  if (!a || a->rows < 0 || a->rows >= (int64_t)1 << 31 || a->vocab < 1 || a->vocab >= (int64_t)1 << 31 || a->inner < 1 ||
      (a->token_bytes != 4 && a->token_bytes != 8) || !(a->temperature > 0.0f) || a->temperature > 3e38f)
    return "token_logprobs: bad arguments";
  if (!known_dtype(a->dtype)) return "token_logprobs: float32 and bfloat16 logits are supported";
  if (a->rows * parts_of<true>(a->vocab * bytes_of(a->dtype)) >= (int64_t)1 << 33) return "token_logprobs: too many logits";   // 2^31 CTAs of eight warps: 32 TB
  if (a->rows && (!a->logits || !a->tokens || reinterpret_cast<uintptr_t>(a->stats) % 8)) return "token_logprobs: null or unaligned pointer";
  return nullptr;
}
Args args_of(const advopt_token_logprobs_args& a, int64_t parts) {
  const double inv = 1.0 / (double)a.temperature;
  return {a.logprobs, a.stats, static_cast<float2*>(a.work), a.logits, a.tokens, a.err, a.inner, a.ld_outer, a.ld_inner, a.rows, a.ignore, (uint32_t)a.vocab,
          (uint32_t)parts,          a.token_bytes == 8, (float)(inv * 1.4426950408889634), (float)inv};
}

}  // namespace lp
}  // namespace advopt

using namespace advopt;

extern "C" int64_t advopt_token_logprobs_work(int64_t rows, int64_t vocab, int32_t dtype) {
  const int64_t parts = rows <= 0 || vocab <= 0 ? 0 : lp::parts_of<false>(vocab * bytes_of(dtype));
  return parts > 1 && !lp::alone(rows, parts) ? rows * parts * 8 : 0;
}

extern "C" int advopt_token_logprobs(const advopt_token_logprobs_args* a, void* stream) {
  if (const char* why = lp::check(a)) return set_error(ADVOPT_E_INVALID, why);
  if (a->rows == 0) return ADVOPT_OK;
  if (!a->logprobs || (advopt_token_logprobs_work(a->rows, a->vocab, a->dtype) && (!a->work || reinterpret_cast<uintptr_t>(a->work) % 8)))
    return set_error(ADVOPT_E_INVALID, "token_logprobs: null output or workspace");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const lp::Args q = lp::args_of(*a, lp::parts_of<false>(a->vocab * bytes_of(a->dtype)));
  return check_cuda(a->dtype == ADVOPT_DT_BF16 ? lp::forward<true>(q, s) : lp::forward<false>(q, s), "advopt_token_logprobs");
}

extern "C" int advopt_token_logprobs_grad(void* dlogits, const float* dlogprobs, const advopt_token_logprobs_args* a, void* stream) {
  if (const char* why = lp::check(a)) return set_error(ADVOPT_E_INVALID, why);
  if (a->rows == 0) return ADVOPT_OK;
  if (!dlogits || !aligned16(dlogits) || !dlogprobs || !a->stats)
    return set_error(ADVOPT_E_INVALID, "token_logprobs_grad: null or unaligned pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const lp::Args q = lp::args_of(*a, lp::parts_of<true>(a->vocab * bytes_of(a->dtype)));
  return check_cuda(a->dtype == ADVOPT_DT_BF16 ? lp::grad<true>(dlogits, dlogprobs, q, s) : lp::grad<false>(dlogits, dlogprobs, q, s),
                    "advopt_token_logprobs_grad");
}
