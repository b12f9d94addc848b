// Layer norm: y = (x - mean) * rstd * w + b over rows, and its gradients
//   g = dy * w, h = (x - mean) * rstd,
//   dx = rstd * (g - mean of g - h * mean of g h), dw = sum of dy h, db = sum of dy.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and
// writes dx, each once.  A row stays in the registers of one warp (up to 1024
// columns) or one CTA (up to 8192), so the variance is that of the
// differences from the mean, in float32, without a second read.  Wider rows
// are read again (from L2).  dw and db are summed down the columns that a
// thread holds, over all rows its CTA takes; the CTAs' sums are added in order
// by a second launch, so that results repeat bit for bit.
#include <atomic>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace advopt {
namespace ln {

constexpr int WARPS = 8;      // rows at a time of a CTA whose warps take a row each

// Sums of N values over the warp or the CTA; every thread gets them.  `red` has
// room for two rounds, so that one barrier a round is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[32 * N], int& round) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (!WARP) {
    const int warps = blockDim.x >> 5;
    float* r = red[round & 1];
    ++round;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[(threadIdx.x >> 5) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
    for (int w = 0; w < warps; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], r[w * N + i]);
    }
  }
}

template <int NV>
__device__ __forceinline__ void columns(int64_t cols, int width, int lane, int64_t (&c)[NV], int (&nv)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    c[v] = ((int64_t)v * width + lane) * 8;
    nv[v] = c[v] >= cols ? 0 : cols - c[v] < 8 ? (int)(cols - c[v]) : 8;
  }
}

// Eight weights, or `absent` where there are none.
template <bool BW>
__device__ __forceinline__ void weights(Oct<BW>& w, const void* p, float absent, int64_t c, int nv, bool vec) {
  if (p) {
    w.get(p, c, nv, vec);
  } else {
    const float v[8] = {absent, absent, absent, absent, absent, absent, absent, absent};
    w.set(v);
  }
}

// ---- rows on their way through shared memory ----
// A thread copies the 16-byte granules that it will read itself, several rows
// ahead, so that only its own copies have to be waited for.  Rows that do not
// start on a 16-byte boundary (A false) are copied from the boundary before:
// every granule holds an element of the row, and a thread's eight elements
// then reach into the granule behind its own, which is the next lane's (the
// last lane copies it too).
template <bool BF16, int NV, bool A, int S>
struct Rows {
  static constexpr int G = BF16 ? 1 : 2;            // granules of eight elements
  static constexpr int SIZE = BF16 ? 2 : 4;
  uint4* slots;                                     // [S][NV][G][threads], then [S][NV][warps]
  const unsigned char* base;
  int64_t pitch;                                    // bytes
  int64_t bytes;                                    // of a row
  uint32_t first[NV];                               // this thread's first granules

  // 16-byte slots of a CTA
  __host__ __device__ static constexpr int slots_of(int threads) { return S * NV * (G * threads + (A ? 0 : threads / 32)); }
  __device__ __forceinline__ uint4* own(int s, int v, int g) const { return slots + ((s * NV + v) * G + g) * blockDim.x + threadIdx.x; }
  __device__ __forceinline__ uint4* last(int s, int v) const {
    return slots + S * NV * G * blockDim.x + (s * NV + v) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  }
  __device__ __forceinline__ static void copy(uint4* to, const unsigned char* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  }
  __device__ __forceinline__ void init(uint4* smem, const void* p, int64_t ld, int64_t cols, const int64_t (&c)[NV]) {
    slots = smem;
    base = static_cast<const unsigned char*>(p);
    pitch = ld * SIZE;
    bytes = cols * SIZE;
#pragma unroll
    for (int v = 0; v < NV; ++v) first[v] = (uint32_t)(c[v] / 8 * G);
  }
  __device__ __forceinline__ uint32_t off(int64_t r) const { return A ? 0u : (uint32_t)reinterpret_cast<uintptr_t>(base + r * pitch) & 15u; }
  __device__ __forceinline__ void issue(int64_t r, int s) const {
    const uint32_t o = off(r);
    const unsigned char* p = base + r * pitch - o;
    const int64_t end = bytes + o;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int64_t at = (int64_t)(first[v] + g) * 16;
        if (at < end) copy(own(s, v, g), p + at);
      }
      if (!A && (threadIdx.x & 31) == 31) {
        const int64_t at = (int64_t)(first[v] + G) * 16;
        if (at < end) copy(last(s, v), p + at);
      }
    }
  }
  // Row r's elements, zeros behind its end.  All lanes take part; the copies have been waited for.
  __device__ __forceinline__ void get(Oct<BF16>& x, int64_t r, int s, int v, int nv) const {
    uint4 q[G + 1];
#pragma unroll
    for (int g = 0; g < G; ++g) q[g] = *own(s, v, g);
    if (A) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        x.w[4 * g] = q[g].x; x.w[4 * g + 1] = q[g].y; x.w[4 * g + 2] = q[g].z; x.w[4 * g + 3] = q[g].w;
      }
    } else {
      q[G] = (threadIdx.x & 31) == 31 ? *last(s, v) : *(own(s, v, 0) + 1);
      const uint32_t o = off(r);
      const bool by8 = o & 8, by4 = o & 4, by2 = o & 2;
      uint32_t t[4 * G + 4];
#pragma unroll
      for (int g = 0; g <= G; ++g) {
        t[4 * g] = q[g].x; t[4 * g + 1] = q[g].y; t[4 * g + 2] = q[g].z; t[4 * g + 3] = q[g].w;
      }
#pragma unroll
      for (int i = 0; i < 4 * G + 2; ++i) t[i] = by8 ? t[i + 2] : t[i];
#pragma unroll
      for (int i = 0; i < 4 * G + 1; ++i) t[i] = by4 ? t[i + 1] : t[i];
#pragma unroll
      for (int i = 0; i < 4 * G; ++i) x.w[i] = BF16 && by2 ? __funnelshift_r(t[i], t[i + 1], 16) : t[i];
    }
    if (nv < 8) {
#pragma unroll
      for (int i = 0; i < Oct<BF16>::kWords; ++i) {
        if (BF16) x.w[i] &= (2 * i < nv ? 0xFFFFu : 0u) | (2 * i + 1 < nv ? 0xFFFF0000u : 0u);
        else x.w[i] = i < nv ? x.w[i] : 0u;
      }
    }
  }
};
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Eight elements at column c of an output row.  Where rows do not start on
// 16-byte boundaries (A false), a lane stores the granule that its elements
// begin in, with the lane before's last ones, and by itself only elements whose
// granule no lane has whole.  All lanes take part.
template <bool BF16, bool A>
__device__ __forceinline__ void put_row(const Oct<BF16>& x, void* row, int64_t c, int nv, int64_t cols) {
  if (A) {
    if (nv) x.store(row, c);
    return;
  }
  constexpr int SIZE = BF16 ? 2 : 4, PER = 16 / SIZE, W = Oct<BF16>::kWords;
  unsigned char* p = static_cast<unsigned char*>(row) + c * SIZE;
  const uint32_t o = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const int k = (int)o / SIZE, lane = threadIdx.x & 31;
  // words: the previous lane's last four, then this lane's
  uint32_t t[4 + W];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __shfl_up_sync(0xffffffffu, x.w[W - 4 + i], 1);
#pragma unroll
  for (int i = 0; i < W; ++i) t[4 + i] = x.w[i];
  const bool whole = lane > 0 && nv == 8, next = lane < 31 && c + 16 <= cols;
  if (nv == 8) {
    // the granules from p - o on: words of t from byte 16 - o on
    const uint32_t back = (16u - o) & 15u;
    uint32_t u[W + 2];
    const bool by16 = o == 0, by8 = back & 8, by4 = back & 4, by2 = back & 2;
#pragma unroll
    for (int i = 0; i < W + 2; ++i) u[i] = by8 ? t[i + 2 < 4 + W ? i + 2 : 3 + W] : t[i];
#pragma unroll
    for (int i = 0; i < W + 1; ++i) u[i] = by4 ? u[i + 1] : u[i];
    uint32_t g[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      g[i] = BF16 && by2 ? __funnelshift_r(u[i], u[i + 1], 16) : u[i];
      if (by16) g[i] = x.w[i];
    }
    uint4* to = reinterpret_cast<uint4*>(p - o);
    if (whole || by16) to[0] = make_uint4(g[0], g[1], g[2], g[3]);
    if constexpr (!BF16) to[1] = make_uint4(g[W - 4], g[W - 3], g[W - 2], g[W - 1]);
    if (by16) return;
  }
  // one by one: those of the first granule where it is not whole, those behind the last one where the next lane does not store them
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool early = nv == 8 ? e < PER - k && !whole : e < 8 - k;
    const bool late = e >= 8 - k && !next;
    if (e < nv && (early || late)) {
      if (BF16) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(x.w[(e >> 1) & (W - 1)] >> (16 * (e & 1)));
      else reinterpret_cast<uint32_t*>(p)[e] = x.w[e & (W - 1)];
    }
  }
}

constexpr int FWD_STAGES = 4, GRAD_STAGES = 3;

template <bool BX, bool BW, int NV, bool WARP, bool A>
__global__ void __launch_bounds__(WARP ? WARPS * 32 : 512) forward_kernel(const __grid_constant__ advopt_layer_norm_args a, int wvec) {
  extern __shared__ uint4 smem[];
  __shared__ float red[2][32];
  const int width = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  int64_t c[NV];
  int nv[NV];
  columns<NV>(a.cols, width, lane, c, nv);
  constexpr int S = FWD_STAGES;
  Rows<BX, NV, A, S> rows;
  rows.init(smem, a.x, a.ldx, a.cols, c);
  const int64_t step = (int64_t)gridDim.x * (WARP ? WARPS : 1);
  int64_t r = WARP ? (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    if (r + s * step < a.rows) rows.issue(r + s * step, s);
    commit_copies();
  }
  Oct<BW> w[NV], b[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    weights(w[v], a.weight, 1.0f, c[v], nv[v], wvec);
    weights(b[v], a.bias, 0.0f, c[v], nv[v], wvec);
  }
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  int round = 0, stage = 0;
  for (; r < a.rows; r += step) {
    wait_copies<S - 2>();
    if (!A) __syncwarp();   // the next lane's copies are read too
    Oct<BX> x[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) rows.get(x[v], r, stage, v, nv[v]);
    if (!A) __syncwarp();
    // into the stage that was read a row ago
    const int free = stage == 0 ? S - 1 : stage - 1;
    if (r + (S - 1) * step < a.rows) rows.issue(r + (S - 1) * step, free);
    commit_copies();
    stage = stage == S - 1 ? 0 : stage + 1;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add2(s, x[v].pair(i));   // zeros behind the row's end
    float t[1] = {__fadd_rn(s.x, s.y)};
    row_sum<WARP, 1>(t, red, round);
    const float mean = __fmul_rn(t[0], inv);
    s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 d = add2(x[v].pair(i), splat2(-mean));
        if (nv[v] == 8) {
          s = fma2(d, d, s);
        } else {
          if (2 * i < nv[v]) s.x = __fmaf_rn(d.x, d.x, s.x);
          if (2 * i + 1 < nv[v]) s.y = __fmaf_rn(d.y, d.y, s.y);
        }
      }
    t[0] = __fadd_rn(s.x, s.y);
    row_sum<WARP, 1>(t, red, round);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(t[0], inv, a.eps)));
    if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(mean, rstd);
    unsigned char* to = static_cast<unsigned char*>(a.y) + r * a.cols * (BX ? 2 : 4);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 h = mul2(add2(x[v].pair(i), splat2(-mean)), splat2(rstd));
        h = fma2(h, w[v].pair(i), b[v].pair(i));
        y[2 * i] = h.x;
        y[2 * i + 1] = h.y;
      }
      Oct<BX> o;
      o.set(y);
      put_row<BX, A>(o, to, c[v], nv[v], a.cols);
    }
  }
}

// Rows that no CTA's registers hold: read three times.
template <bool BX, bool BW>
__global__ void __launch_bounds__(1024) wide_forward_kernel(const __grid_constant__ advopt_layer_norm_args a, int vec, int wvec) {
  __shared__ float red[2][32];
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  int round = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    float t[1] = {0.0f};
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      Oct<BX> x;
      x.get(a.x, r * a.ldx + c, a.cols - c < 8 ? (int)(a.cols - c) : 8, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[0] = __fadd_rn(t[0], x.at(e));
    }
    row_sum<false, 1>(t, red, round);
    const float mean = __fmul_rn(t[0], inv);
    t[0] = 0.0f;
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      const int nv = a.cols - c < 8 ? (int)(a.cols - c) : 8;
      Oct<BX> x;
      x.get(a.x, r * a.ldx + c, nv, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = __fsub_rn(x.at(e), mean);
        if (e < nv) t[0] = __fmaf_rn(d, d, t[0]);
      }
    }
    row_sum<false, 1>(t, red, round);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(t[0], inv, a.eps)));
    if (a.stats && threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(mean, rstd);
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      const int nv = a.cols - c < 8 ? (int)(a.cols - c) : 8;
      Oct<BX> x, o;
      Oct<BW> w, b;
      x.get(a.x, r * a.ldx + c, nv, vec);
      weights(w, a.weight, 1.0f, c, nv, wvec);
      weights(b, a.bias, 0.0f, c, nv, wvec);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __fmaf_rn(__fmul_rn(__fsub_rn(x.at(e), mean), rstd), w.at(e), b.at(e));
      o.set(y);
      o.put(a.y, r * a.cols + c, nv, vec);
    }
  }
}

// ---- the gradients ----
template <bool BX, bool BW, int NV, bool WARP, bool A>
__global__ void __launch_bounds__(WARP ? WARPS * 32 : 512) grad_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int wvec) {
  extern __shared__ uint4 smem[];
  __shared__ float red[2][64];
  const int width = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  int64_t c[NV];
  int nv[NV];
  columns<NV>(a.cols, width, lane, c, nv);
  const bool sums = a.work != nullptr;
  constexpr int S = GRAD_STAGES;
  using R = Rows<BX, NV, A, S>;
  R xs, dys;
  xs.init(smem, a.x, a.ldx, a.cols, c);
  dys.init(smem + R::slots_of(blockDim.x), a.dy, a.lddy, a.cols, c);
  const int64_t step = (int64_t)gridDim.x * (WARP ? WARPS : 1);
  int64_t r = WARP ? (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    if (r + s * step < a.rows) {
      xs.issue(r + s * step, s);
      dys.issue(r + s * step, s);
    }
    commit_copies();
  }
  Oct<BW> w[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) weights(w[v], a.weight, 1.0f, c[v], nv[v], wvec);
  float2 dw[NV][4], db[NV][4];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[v][i] = db[v][i] = make_float2(0.0f, 0.0f);
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  int round = 0, stage = 0;
  for (; r < a.rows; r += step) {
    const float2 st = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * r));
    wait_copies<S - 2>();
    if (!A) __syncwarp();   // the next lane's copies are read too
    Oct<BX> x[NV], dy[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xs.get(x[v], r, stage, v, nv[v]);
      dys.get(dy[v], r, stage, v, nv[v]);
    }
    if (!A) __syncwarp();
    // into the stage that was read a row ago
    const int free = stage == 0 ? S - 1 : stage - 1;
    if (r + (S - 1) * step < a.rows) {
      xs.issue(r + (S - 1) * step, free);
      dys.issue(r + (S - 1) * step, free);
    }
    commit_copies();
    stage = stage == S - 1 ? 0 : stage + 1;
    const float mean = st.x, rstd = st.y;
    float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 h = mul2(add2(x[v].pair(i), splat2(-mean)), splat2(rstd)), d = dy[v].pair(i);
        const float2 g = mul2(d, w[v].pair(i));
        s1 = add2(s1, g);   // dy is 0 behind the row's end; h, of a mean that may be infinite, is left out there
        if (nv[v] == 8) {
          s2 = fma2(g, h, s2);
          dw[v][i] = fma2(d, h, dw[v][i]);
        } else {
          if (2 * i < nv[v]) s2.x = __fmaf_rn(g.x, h.x, s2.x), dw[v][i].x = __fmaf_rn(d.x, h.x, dw[v][i].x);
          if (2 * i + 1 < nv[v]) s2.y = __fmaf_rn(g.y, h.y, s2.y), dw[v][i].y = __fmaf_rn(d.y, h.y, dw[v][i].y);
        }
        db[v][i] = add2(db[v][i], d);
      }
    }
    if (!a.dx) continue;
    float t[2] = {__fadd_rn(s1.x, s1.y), __fadd_rn(s2.x, s2.y)};
    row_sum<WARP, 2>(t, red, round);
    const float m1 = __fmul_rn(t[0], inv), m2 = __fmul_rn(t[1], inv);
    unsigned char* to = static_cast<unsigned char*>(a.dx) + r * a.cols * (BX ? 2 : 4);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 h = mul2(add2(x[v].pair(i), splat2(-mean)), splat2(rstd)), d = dy[v].pair(i);
        const float2 g = mul2(d, w[v].pair(i));
        const float2 q = mul2(fma2(h, splat2(-m2), add2(g, splat2(-m1))), splat2(rstd));
        o[2 * i] = q.x;
        o[2 * i + 1] = q.y;
      }
      Oct<BX> oct;
      oct.set(o);
      put_row<BX, A>(oct, to, c[v], nv[v], a.cols);
    }
  }
  if (!sums) return;
  float* part = static_cast<float*>(a.work) + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (WARP) {
    // the warps' sums, a warp's after the other's, in shared memory
    wait_copies<0>();
    __syncthreads();
    float* sh = reinterpret_cast<float*>(smem);   // [2][NV * 256]
    for (int k = 0; k < WARPS; ++k) {
      if ((int)(threadIdx.x >> 5) == k) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* p = sh + c[v] + e;
            const float x0 = e & 1 ? dw[v][e >> 1].y : dw[v][e >> 1].x, x1 = e & 1 ? db[v][e >> 1].y : db[v][e >> 1].x;
            p[0] = k ? __fadd_rn(p[0], x0) : x0;
            p[NV * 256] = k ? __fadd_rn(p[NV * 256], x1) : x1;
          }
      }
      __syncthreads();
    }
    for (int64_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
      part[i] = sh[i];
      part[a.cols + i] = sh[NV * 256 + i];
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < nv[v]) {
          part[c[v] + e] = e & 1 ? dw[v][e >> 1].y : dw[v][e >> 1].x;
          part[a.cols + c[v] + e] = e & 1 ? db[v][e >> 1].y : db[v][e >> 1].x;
        }
  }
}

// Rows that no CTA's registers hold: dx from two reads of a row, dw and db by columns.
template <bool BX, bool BW>
__global__ void __launch_bounds__(1024) wide_dx_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int vec, int wvec) {
  __shared__ float red[2][64];
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  int round = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float mean = __ldg(a.stats + 2 * r), rstd = __ldg(a.stats + 2 * r + 1);
    float t[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      const int nv = a.cols - c < 8 ? (int)(a.cols - c) : 8;
      Oct<BX> x, dy;
      Oct<BW> w;
      x.get(a.x, r * a.ldx + c, nv, vec);
      dy.get(a.dy, r * a.lddy + c, nv, vec);
      weights(w, a.weight, 1.0f, c, nv, wvec);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e >= nv) break;
        const float g = __fmul_rn(dy.at(e), w.at(e));
        t[0] = __fadd_rn(t[0], g);
        t[1] = __fmaf_rn(g, __fmul_rn(__fsub_rn(x.at(e), mean), rstd), t[1]);
      }
    }
    row_sum<false, 2>(t, red, round);
    const float m1 = __fmul_rn(t[0], inv), m2 = __fmul_rn(t[1], inv);
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      const int nv = a.cols - c < 8 ? (int)(a.cols - c) : 8;
      Oct<BX> x, dy, oct;
      Oct<BW> w;
      x.get(a.x, r * a.ldx + c, nv, vec);
      dy.get(a.dy, r * a.lddy + c, nv, vec);
      weights(w, a.weight, 1.0f, c, nv, wvec);
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = __fmul_rn(dy.at(e), w.at(e));
        const float h = __fmul_rn(__fsub_rn(x.at(e), mean), rstd);
        o[e] = __fmul_rn(__fmaf_rn(h, -m2, __fsub_rn(g, m1)), rstd);
      }
      oct.set(o);
      oct.put(a.dx, r * a.cols + c, nv, vec);
    }
  }
}

// A warp: 256 columns, every gridDim.y-th row; one row of partial sums for each blockIdx.y.
template <bool BX>
__global__ void __launch_bounds__(256) wide_sums_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int vec) {
  __shared__ float sh[2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8;
  const int nv = c >= a.cols ? 0 : a.cols - c < 8 ? (int)(a.cols - c) : 8;
  float dw[8] = {}, db[8] = {};
  for (int64_t r = (int64_t)blockIdx.y * 8 + warp; r < a.rows; r += (int64_t)gridDim.y * 8) {
    const float mean = __ldg(a.stats + 2 * r), rstd = __ldg(a.stats + 2 * r + 1);
    Oct<BX> x, dy;
    x.get(a.x, r * a.ldx + c, nv, vec);
    dy.get(a.dy, r * a.lddy + c, nv, vec);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= nv) break;
      dw[e] = __fmaf_rn(dy.at(e), __fmul_rn(__fsub_rn(x.at(e), mean), rstd), dw[e]);
      db[e] = __fadd_rn(db[e], dy.at(e));
    }
  }
  for (int k = 0; k < 8; ++k) {
    if (warp == k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sh[0][lane * 8 + e] = k ? __fadd_rn(sh[0][lane * 8 + e], dw[e]) : dw[e];
        sh[1][lane * 8 + e] = k ? __fadd_rn(sh[1][lane * 8 + e], db[e]) : db[e];
      }
    }
    __syncthreads();
  }
  float* part = static_cast<float*>(a.work) + (int64_t)blockIdx.y * 2 * a.cols;
  const int64_t mine = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (mine < a.cols) {
    part[mine] = sh[0][threadIdx.x];
    part[a.cols + mine] = sh[1][threadIdx.x];
  }
}

// dweight and dbias from the CTAs' sums: 32 columns a CTA, the parts split over its warps in order.
constexpr int FINISH_WARPS = 16;
template <bool BW>
__global__ void __launch_bounds__(FINISH_WARPS * 32) finish_kernel(void* dweight, void* dbias, const float* part, int64_t parts, int64_t cols) {
  __shared__ float red[FINISH_WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  void* out = blockIdx.y ? dbias : dweight;
  const float* p = part + blockIdx.y * cols + c;
  const int64_t each = (parts + FINISH_WARPS - 1) / FINISH_WARPS;
  const int64_t begin = warp * each, end = begin + each < parts ? begin + each : parts;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t i = begin; i < end; ++i) s = __fadd_rn(s, __ldg(p + i * 2 * cols));
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols && out) {
    s = red[0][lane];
#pragma unroll
    for (int w = 1; w < FINISH_WARPS; ++w) s = __fadd_rn(s, red[w][lane]);
    if (BW) static_cast<uint16_t*>(out)[c] = (uint16_t)f_to_bf16_rne(s);
    else static_cast<float*>(out)[c] = s;
  }
}

// ---- variants ----
constexpr int64_t MOST = 8192;      // columns that a CTA's registers hold
constexpr int64_t WARP_MOST = 1024; // and a warp's
constexpr int64_t SMS = 148;

inline int block_threads(int64_t cols) { return (int)ceil_div(cols, 2 * 8 * 32) * 32; }
// CTAs of the gradient kernel at most: each leaves a row of partial sums, so a CTA takes four rows at least where that leaves one for each SM.
inline int64_t grad_ctas(int64_t rows, int64_t cols) {
  const int64_t units = cols <= WARP_MOST ? ceil_div(rows, WARPS) : rows;
  const int64_t few = ceil_div(units, 4) > SMS ? ceil_div(units, 4) : SMS, most = 8 * SMS;
  const int64_t n = few < most ? few : most;
  return units < n ? units : n;
}
inline int64_t wide_parts(int64_t rows) { return rows < 8 * 32 ? ceil_div(rows, 8) : 32; }

// Launches a persistent kernel with as many CTAs as fit the SMs, `most` at most; the number of CTAs, or -1.
template <auto KERNEL, class Arg>
int64_t launch(const Arg& a, int wvec, int threads, int smem, int64_t most, cudaStream_t s) {
  static std::atomic<int> resident[33];   // this kernel's, by warps
  // for the current device, whichever that is
  if (smem > 47 * 1024 && cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -1;
  int n = resident[threads / 32].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, smem) != cudaSuccess || n < 1) return -1;
    resident[threads / 32].store(n, std::memory_order_relaxed);
  }
  const int64_t grid = n * SMS < most ? n * SMS : most;
  KERNEL<<<(unsigned)grid, threads, smem, s>>>(a, wvec);
  return grid;
}

template <bool BX, bool BW, int NV, bool WARP>
int64_t forward_variant(const advopt_layer_norm_args& a, bool vec, int wvec, cudaStream_t s) {
  const int threads = WARP ? WARPS * 32 : block_threads(a.cols);
  const int64_t most = WARP ? ceil_div(a.rows, WARPS) : a.rows;
  if (vec) return launch<forward_kernel<BX, BW, NV, WARP, true>>(a, wvec, threads, Rows<BX, NV, true, FWD_STAGES>::slots_of(threads) * 16, most, s);
  return launch<forward_kernel<BX, BW, NV, WARP, false>>(a, wvec, threads, Rows<BX, NV, false, FWD_STAGES>::slots_of(threads) * 16, most, s);
}

template <bool BX, bool BW>
int forward(const advopt_layer_norm_args& a, cudaStream_t s) {
  const bool vec = aligned16(a.x) && aligned16(a.y) && a.cols % 8 == 0 && a.ldx * (BX ? 2 : 4) % 16 == 0;
  const int wvec = aligned16(a.weight) && aligned16(a.bias);
  int64_t n = 1;
  if (a.cols > MOST) wide_forward_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
  else if (a.cols <= 256) n = forward_variant<BX, BW, 1, true>(a, vec, wvec, s);
  else if (a.cols <= 512) n = forward_variant<BX, BW, 2, true>(a, vec, wvec, s);
  else if (a.cols <= WARP_MOST) n = forward_variant<BX, BW, 4, true>(a, vec, wvec, s);
  else n = forward_variant<BX, BW, 2, false>(a, vec, wvec, s);
  const cudaError_t e = cudaGetLastError();
  return n < 0 ? set_error(ADVOPT_E_CUDA, "advopt_layer_norm: the kernel's attributes") : check_cuda(e, "advopt_layer_norm");
}

template <bool BX, bool BW, int NV, bool WARP>
int64_t grad_variant(const advopt_layer_norm_grad_args& a, bool vec, int wvec, cudaStream_t s) {
  const int threads = WARP ? WARPS * 32 : block_threads(a.cols);
  const int64_t most = grad_ctas(a.rows, a.cols);
  if (vec) return launch<grad_kernel<BX, BW, NV, WARP, true>>(a, wvec, threads, 2 * Rows<BX, NV, true, GRAD_STAGES>::slots_of(threads) * 16, most, s);
  return launch<grad_kernel<BX, BW, NV, WARP, false>>(a, wvec, threads, 2 * Rows<BX, NV, false, GRAD_STAGES>::slots_of(threads) * 16, most, s);
}

template <bool BX, bool BW>
int grad(const advopt_layer_norm_grad_args& a, cudaStream_t s) {
  const bool vec = aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) && a.cols % 8 == 0 && a.ldx * (BX ? 2 : 4) % 16 == 0 &&
                   a.lddy * (BX ? 2 : 4) % 16 == 0;
  const int wvec = aligned16(a.weight);
  int64_t parts = 0;
  if (a.cols > MOST) {
    parts = wide_parts(a.rows);
    if (a.dx) wide_dx_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
    if (a.work) wide_sums_kernel<BX><<<dim3((unsigned)ceil_div(a.cols, 256), (unsigned)parts), 256, 0, s>>>(a, vec);
  } else if (a.cols <= 256) {
    parts = grad_variant<BX, BW, 1, true>(a, vec, wvec, s);
  } else if (a.cols <= 512) {
    parts = grad_variant<BX, BW, 2, true>(a, vec, wvec, s);
  } else if (a.cols <= WARP_MOST) {
    parts = grad_variant<BX, BW, 4, true>(a, vec, wvec, s);
  } else {
    parts = grad_variant<BX, BW, 2, false>(a, vec, wvec, s);
  }
  if (parts > 0 && a.work)
    finish_kernel<BW><<<dim3((unsigned)ceil_div(a.cols, 32), 2), FINISH_WARPS * 32, 0, s>>>(a.dweight, a.dbias, static_cast<const float*>(a.work),
                                                                                            parts, a.cols);
  const cudaError_t e = cudaGetLastError();
  return parts < 0 ? set_error(ADVOPT_E_CUDA, "advopt_layer_norm_grad: the kernel's attributes") : check_cuda(e, "advopt_layer_norm_grad");
}

constexpr int64_t LIMIT = (int64_t)1 << 31;

}  // namespace ln
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_layer_norm(const advopt_layer_norm_args* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 0 || a->rows >= ((int64_t)1 << 40) || a->cols >= ln::LIMIT || (a->rows > 1 && a->ldx < a->cols) ||
      !(a->eps >= 0.0f))
    return set_error(ADVOPT_E_INVALID, "advopt_layer_norm: bad arguments");
  if (!known_dtype(a->x_dtype) || !known_dtype(a->w_dtype))
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_layer_norm: float32 and bfloat16 are supported");
  if (a->rows == 0 || a->cols == 0) return ADVOPT_OK;
  if (!a->x || !a->y || reinterpret_cast<uintptr_t>(a->stats) % 8)
    return set_error(ADVOPT_E_INVALID, "advopt_layer_norm: null or unaligned pointer");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bx = a->x_dtype == ADVOPT_DT_BF16, bw = a->w_dtype == ADVOPT_DT_BF16;
  return bx ? bw ? ln::forward<true, true>(*a, s) : ln::forward<true, false>(*a, s)
            : bw ? ln::forward<false, true>(*a, s) : ln::forward<false, false>(*a, s);
}

extern "C" int64_t advopt_layer_norm_grad_work(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (cols > ln::MOST ? ln::wide_parts(rows) : ln::grad_ctas(rows, cols)) * 2 * cols * 4;
}

extern "C" int advopt_layer_norm_grad(const advopt_layer_norm_grad_args* a, void* stream) {
  if (!a || a->rows < 0 || a->cols < 0 || a->rows >= ((int64_t)1 << 40) || a->cols >= ln::LIMIT ||
      (a->rows > 1 && (a->ldx < a->cols || a->lddy < a->cols)))
    return set_error(ADVOPT_E_INVALID, "advopt_layer_norm_grad: bad arguments");
  if (!known_dtype(a->x_dtype) || !known_dtype(a->w_dtype))
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_layer_norm_grad: float32 and bfloat16 are supported");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wanted = a->dweight || a->dbias;
  if (a->cols == 0 || (!a->dx && !wanted)) return ADVOPT_OK;
  if (a->rows == 0) {
    const size_t bytes = (size_t)a->cols * bytes_of(a->w_dtype);
    cudaError_t e = a->dweight ? cudaMemsetAsync(a->dweight, 0, bytes, s) : cudaSuccess;
    if (e == cudaSuccess && a->dbias) e = cudaMemsetAsync(a->dbias, 0, bytes, s);
    return check_cuda(e, "advopt_layer_norm_grad");
  }
  if (!a->x || !a->dy || !a->stats || reinterpret_cast<uintptr_t>(a->stats) % 8 || (wanted && (!a->work || !aligned16(a->work))))
    return set_error(ADVOPT_E_INVALID, "advopt_layer_norm_grad: null or unaligned pointer");
  advopt_layer_norm_grad_args q = *a;
  if (!wanted) q.work = nullptr;
  const bool bx = a->x_dtype == ADVOPT_DT_BF16, bw = a->w_dtype == ADVOPT_DT_BF16;
  return bx ? bw ? ln::grad<true, true>(q, s) : ln::grad<true, false>(q, s)
            : bw ? ln::grad<false, true>(q, s) : ln::grad<false, false>(q, s);
}
