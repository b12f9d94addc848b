// Layer norm: y = (x - mean) * rstd * w + b over rows, and its gradients
//   g = dy * w, h = (x - mean) * rstd,
//   dx = rstd * (g - mean of g - h * mean of g h), dw = sum of dy h, db = sum of dy.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and
// writes dx, each once.  A row stays in the registers of one warp (up to 1024
// columns) or one CTA (up to 8192 or 16384), so the variance is that of the
// differences from the mean, in float32, without a second read.  Wider rows
// are read again (from L2).  dw and db are summed down the columns that a
// thread holds, over all rows its CTA takes; the CTAs' sums are added in order
// by a second launch, so that results repeat bit for bit.
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

template <bool BX, bool BW, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? WARPS * 32 : 1024)
    forward_kernel(const __grid_constant__ advopt_layer_norm_args a, int vec, int wvec) {
  __shared__ float red[2][32];
  const int width = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  int64_t c[NV];
  int nv[NV];
  columns<NV>(a.cols, width, lane, c, nv);
  Oct<BW> w[NV], b[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    weights(w[v], a.weight, 1.0f, c[v], nv[v], wvec);
    weights(b[v], a.bias, 0.0f, c[v], nv[v], wvec);
  }
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  const int64_t step = (int64_t)gridDim.x * (WARP ? WARPS : 1);
  int round = 0;
  for (int64_t r = WARP ? (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5) : (int64_t)blockIdx.x; r < a.rows; r += step) {
    Oct<BX> x[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v].get(a.x, r * a.ldx + c[v], nv[v], vec);
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
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (nv[v] == 0) continue;
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
      o.put(a.y, r * a.cols + c[v], nv[v], vec);
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
template <bool BX, bool BW, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? WARPS * 32 : 1024)
    grad_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int vec, int wvec) {
  __shared__ float red[2][64];
  const int width = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  int64_t c[NV];
  int nv[NV];
  columns<NV>(a.cols, width, lane, c, nv);
  const bool sums = a.work != nullptr;
  Oct<BW> w[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) weights(w[v], a.weight, 1.0f, c[v], nv[v], wvec);
  float2 dw[NV][4], db[NV][4];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[v][i] = db[v][i] = make_float2(0.0f, 0.0f);
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  const int64_t step = (int64_t)gridDim.x * (WARP ? WARPS : 1);
  int round = 0;
  for (int64_t r = WARP ? (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5) : (int64_t)blockIdx.x; r < a.rows; r += step) {
    Oct<BX> x[NV], dy[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x[v].get(a.x, r * a.ldx + c[v], nv[v], vec);
      dy[v].get(a.dy, r * a.lddy + c[v], nv[v], vec);
    }
    const float2 st = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * r));
    const float mean = st.x, rstd = st.y;
    float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (nv[v] == 0) continue;   // dy is 0 behind the row's end, so x may be anything finite there
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 h = mul2(add2(x[v].pair(i), splat2(-mean)), splat2(rstd)), d = dy[v].pair(i);
        const float2 g = mul2(d, w[v].pair(i));
        s1 = add2(s1, g);
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
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (nv[v] == 0) continue;
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
      oct.put(a.dx, r * a.cols + c[v], nv[v], vec);
    }
  }
  if (!sums) return;
  float* part = static_cast<float*>(a.work) + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (WARP) {
    // the warps' sums, a warp's after the other's, in shared memory
    extern __shared__ float sh[];   // [2][NV * 256]
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
constexpr int64_t FWD_MOST = 16384, GRAD_MOST = 8192;   // columns that a CTA's registers hold
constexpr int64_t SMS = 148;

// CTAs of the gradient kernel, each of which leaves a row of partial sums.
inline int64_t grad_ctas(int64_t rows, int64_t cols) {
  const int64_t units = cols <= 1024 ? ceil_div(rows, WARPS) : rows;
  const int64_t most = SMS * (cols <= 1024 ? 2 : cols <= 2048 ? 8 : cols <= 4096 ? 4 : 2);
  return units < most ? units : most;
}
inline int64_t wide_parts(int64_t rows) { return rows < 8 * 32 ? ceil_div(rows, 8) : 32; }

template <bool BX, bool BW>
void forward(const advopt_layer_norm_args& a, cudaStream_t s) {
  const int vec = aligned16(a.x) && aligned16(a.y) && a.cols % 8 == 0 && a.ldx * (BX ? 2 : 4) % 16 == 0;
  const int wvec = aligned16(a.weight) && aligned16(a.bias);
  if (a.cols > FWD_MOST) {
    wide_forward_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
  } else if (a.cols <= 1024) {
    const int64_t ctas = ceil_div(a.rows, WARPS);
    const unsigned grid = (unsigned)(ctas < SMS * 8 ? ctas : SMS * 8);
    if (a.cols <= 256) forward_kernel<BX, BW, 1, true><<<grid, WARPS * 32, 0, s>>>(a, vec, wvec);
    else if (a.cols <= 512) forward_kernel<BX, BW, 2, true><<<grid, WARPS * 32, 0, s>>>(a, vec, wvec);
    else forward_kernel<BX, BW, 4, true><<<grid, WARPS * 32, 0, s>>>(a, vec, wvec);
  } else {
    const int threads = (int)ceil_div(a.cols, 2 * 8 * 32) * 32;
    const int64_t most = SMS * (2048 / threads);
    forward_kernel<BX, BW, 2, false><<<(unsigned)(a.rows < most ? a.rows : most), threads, 0, s>>>(a, vec, wvec);
  }
}

template <bool BX, bool BW>
void grad(const advopt_layer_norm_grad_args& a, cudaStream_t s) {
  const int vec = aligned16(a.x) && aligned16(a.dy) && aligned16(a.dx) && a.cols % 8 == 0 && a.ldx * (BX ? 2 : 4) % 16 == 0 &&
                  a.lddy * (BX ? 2 : 4) % 16 == 0;
  const int wvec = aligned16(a.weight);
  int64_t parts = grad_ctas(a.rows, a.cols);
  if (a.cols > GRAD_MOST) {
    parts = wide_parts(a.rows);
    if (a.dx) wide_dx_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
    if (a.work) wide_sums_kernel<BX><<<dim3((unsigned)ceil_div(a.cols, 256), (unsigned)parts), 256, 0, s>>>(a, vec);
  } else if (a.cols <= 256) {
    grad_kernel<BX, BW, 1, true><<<(unsigned)parts, WARPS * 32, 2 * 256 * 4, s>>>(a, vec, wvec);
  } else if (a.cols <= 512) {
    grad_kernel<BX, BW, 2, true><<<(unsigned)parts, WARPS * 32, 2 * 512 * 4, s>>>(a, vec, wvec);
  } else if (a.cols <= 1024) {
    grad_kernel<BX, BW, 4, true><<<(unsigned)parts, WARPS * 32, 2 * 1024 * 4, s>>>(a, vec, wvec);
  } else {
    grad_kernel<BX, BW, 1, false><<<(unsigned)parts, (unsigned)ceil_div(a.cols, 8 * 32) * 32, 0, s>>>(a, vec, wvec);
  }
  if (a.work)
    finish_kernel<BW><<<dim3((unsigned)ceil_div(a.cols, 32), 2), FINISH_WARPS * 32, 0, s>>>(a.dweight, a.dbias, static_cast<const float*>(a.work),
                                                                                            parts, a.cols);
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
  if (bx && bw) ln::forward<true, true>(*a, s);
  else if (bx) ln::forward<true, false>(*a, s);
  else if (bw) ln::forward<false, true>(*a, s);
  else ln::forward<false, false>(*a, s);
  return check_cuda(cudaGetLastError(), "advopt_layer_norm");
}

extern "C" int64_t advopt_layer_norm_grad_work(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (cols > ln::GRAD_MOST ? ln::wide_parts(rows) : ln::grad_ctas(rows, cols)) * 2 * cols * 4;
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
  if (bx && bw) ln::grad<true, true>(q, s);
  else if (bx) ln::grad<true, false>(q, s);
  else if (bw) ln::grad<false, true>(q, s);
  else ln::grad<false, false>(q, s);
  return check_cuda(cudaGetLastError(), "advopt_layer_norm_grad");
}
