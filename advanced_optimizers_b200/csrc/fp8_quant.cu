// Block quantisation to 8-bit floating point with power-of-two scales.
//
// For a block (1 x 128 along the contraction, or 128 x 128) with largest
// finite magnitude a, the scale is 2^e with e the least integer for which
// a <= fmax 2^e (fmax = 1.75 * 2^8 for E4M3, 1.75 * 2^15 for E5M2), read off
// a's exponent and mantissa bits; x * 2^-e is exact, so a code carries one
// rounding (nearest even).
//
// Bound: HBM (read x once, write one byte per element and layout).
#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "drop.cuh"

namespace advopt {
namespace fp8q {

constexpr int TILE = 128;

// |x|'s bits, 0 for an infinity or NaN (they do not enter a block's scale).
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t a = f2u(x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}

// Biased scale exponent (E8M0 byte) from the block maximum's bits.
template <bool E5M2>
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
  if (a == 0) return 127u;
  const int b = (int)(a >> 23) - (E5M2 ? 15 : 8) + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b > 0 ? (uint32_t)b : 0u;
}
// 2^-e of a scale byte (at most 247, so the exponent field stays normal)
__device__ __forceinline__ float inv_scale(uint32_t byte) { return u2f((254u - byte) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
  uint16_t r;
  if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// x * 2^-e; an infinity becomes NaN (0 * inf), a finite product is unchanged
// (adding 0 of x's sign).
__device__ __forceinline__ float scaled(float x, float inv) { return __fmaf_rn(x, 0.0f, __fmul_rn(x, inv)); }

template <bool E5M2>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inv) {
  return cvt2<E5M2>(scaled(a, inv), scaled(b, inv)) | (cvt2<E5M2>(scaled(c, inv), scaled(d, inv)) << 16);
}

__device__ __forceinline__ void drop8(float (&v)[8], const DropSpec& d, uint32_t step, uint64_t k0) {
  const uint32_t keep = drop_keep<8>(d, step, k0);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (keep >> e) & 1u ? __fmul_rn(v[e], d.scale) : 0.0f;
}

struct QArgs {
  const void* x;
  int64_t ldx, rows, cols;
  uint8_t* codes_r;
  int64_t ld_r;
  uint8_t* scales_r;
  int64_t ld_sr;
  uint8_t* codes_c;
  int64_t ld_c;
  uint8_t* scales_c;
  int64_t ld_sc;
  float* col_partial;
  int vec, drop;
};

// ---- rows only, 1 x 128 blocks: sixteen lanes per block, eight elements a lane ----
template <bool BF16, bool E5M2>
__global__ void __launch_bounds__(256) rows_kernel(QArgs q, DropSpec d) {
  const uint32_t step = q.drop ? drop_step(d) : 0u;
  const int l16 = threadIdx.x & 15;
  const int64_t nb = (q.cols + TILE - 1) / TILE;
  const int64_t units = q.rows * nb;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 16);
  // both halves of a warp take every trip: the shuffles below name all lanes
  for (int64_t u0 = (int64_t)blockIdx.x * (blockDim.x / 16) + ((threadIdx.x >> 5) << 1); u0 < units; u0 += stride) {
    const int64_t u = u0 + ((threadIdx.x >> 4) & 1);
    const bool live = u < units;
    const int64_t r = live ? u / nb : 0, b = live ? u - r * nb : 0;
    const int64_t c0 = b * TILE + l16 * 8;
    const int nv = !live || c0 >= q.cols ? 0 : q.cols - c0 < 8 ? (int)(q.cols - c0) : 8;
    float v[8];
    load8<BF16>(q.x, r * q.ldx + c0, nv, q.vec && nv == 8, v);
    if (q.drop && nv) drop8(v, d, step, (uint64_t)(r * q.cols + c0));
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, finite_bits(v[e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const uint32_t sb = scale_byte<E5M2>(a);
    const float inv = inv_scale(sb);
    if (nv) {
      const uint32_t w0 = code4<E5M2>(v[0], v[1], v[2], v[3], inv), w1 = code4<E5M2>(v[4], v[5], v[6], v[7], inv);
      uint8_t* out = q.codes_r + r * q.ld_r + c0;
      if (nv == 8) {
        *reinterpret_cast<uint2*>(out) = make_uint2(w0, w1);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < nv) out[e] = (uint8_t)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
      }
    }
    if (live && l16 == 0) q.scales_r[r * q.ld_sr + b] = (uint8_t)sb;
  }
}

// ---- one 128 x 128 tile per CTA: any layout, both block shapes, column sums ----
// Thread (g, l) of 16 x 16 holds rows 8g .. 8g+7, columns 8l .. 8l+7.
template <bool BF16, bool E5M2, bool SQUARE>
__global__ void __launch_bounds__(256, 2) tile_kernel(QArgs q, DropSpec d) {
  __shared__ __align__(16) uint32_t red[16][TILE];     // column maxima, then column sums
  __shared__ __align__(16) uint8_t turned[TILE * TILE];
  __shared__ uint32_t col_byte[TILE];
  __shared__ uint32_t warp_max_bits[8];
  const uint32_t step = q.drop ? drop_step(d) : 0u;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t r0 = (int64_t)blockIdx.y * TILE, c0 = (int64_t)blockIdx.x * TILE;
  const int64_t c = c0 + l * 8;
  const int nv = c >= q.cols ? 0 : q.cols - c < 8 ? (int)(q.cols - c) : 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + g * 8 + i;
    const int n = r < q.rows ? nv : 0;
    load8<BF16>(q.x, r * q.ldx + c, n, q.vec && n == 8, v[i]);
  }
  if (q.drop) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + g * 8 + i;
      if (r < q.rows && nv) drop8(v[i], d, step, (uint64_t)(r * q.cols + c));
    }
  }
  uint32_t square_byte = 0;
  if (SQUARE) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) a = max(a, finite_bits(v[i][e]));
    a = __reduce_max_sync(0xffffffffu, a);
    if ((threadIdx.x & 31) == 0) warp_max_bits[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) a = max(a, warp_max_bits[w]);
    square_byte = scale_byte<E5M2>(a);
    if (threadIdx.x == 0) {
      if (q.codes_r) q.scales_r[blockIdx.y * q.ld_sr + blockIdx.x] = (uint8_t)square_byte;
      if (q.codes_c) q.scales_c[blockIdx.x * q.ld_sc + blockIdx.y] = (uint8_t)square_byte;
    }
  }
  if (q.codes_r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + g * 8 + i;
      uint32_t sb = square_byte;
      if (!SQUARE) {
        uint32_t a = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) a = max(a, finite_bits(v[i][e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        sb = scale_byte<E5M2>(a);
        if (l == 0 && r < q.rows) q.scales_r[r * q.ld_sr + blockIdx.x] = (uint8_t)sb;
      }
      if (r < q.rows && nv) {
        const float inv = inv_scale(sb);
        const uint32_t w0 = code4<E5M2>(v[i][0], v[i][1], v[i][2], v[i][3], inv);
        const uint32_t w1 = code4<E5M2>(v[i][4], v[i][5], v[i][6], v[i][7], inv);
        uint8_t* out = q.codes_r + r * q.ld_r + c;
        if (nv == 8) {
          *reinterpret_cast<uint2*>(out) = make_uint2(w0, w1);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < nv) out[e] = (uint8_t)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
        }
      }
    }
  }
  if (q.codes_c) {
    if (!SQUARE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, finite_bits(v[i][e]));
        red[g][l * 8 + e] = a;
      }
      __syncthreads();
      if (threadIdx.x < TILE) {
        uint32_t a = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) a = max(a, red[w][threadIdx.x]);
        const uint32_t sb = scale_byte<E5M2>(a);
        col_byte[threadIdx.x] = sb;
        if (c0 + threadIdx.x < q.cols) q.scales_c[(c0 + threadIdx.x) * q.ld_sc + blockIdx.y] = (uint8_t)sb;
      }
      __syncthreads();
    }
    // column 8l + e of the tile is row 8l + e of `turned`: 16 chunks of 8
    // bytes, chunk g kept at g ^ l so that a half-warp's stores (one chunk
    // each of 16 rows) and its loads (one row's 16 chunks) touch all banks
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float inv = inv_scale(SQUARE ? square_byte : col_byte[l * 8 + e]);
      const uint32_t w0 = code4<E5M2>(v[0][e], v[1][e], v[2][e], v[3][e], inv);
      const uint32_t w1 = code4<E5M2>(v[4][e], v[5][e], v[6][e], v[7][e], inv);
      *reinterpret_cast<uint2*>(turned + (l * 8 + e) * TILE + ((g ^ l) << 3)) = make_uint2(w0, w1);
    }
    __syncthreads();
    const int64_t nr = q.rows - r0 - l * 8;   // rows of x left from this thread's chunk on
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int tc = i * 16 + g;
      if (c0 + tc < q.cols && nr > 0) {
        const uint2 w = *reinterpret_cast<const uint2*>(turned + tc * TILE + ((l ^ (tc >> 3)) << 3));
        uint8_t* out = q.codes_c + (c0 + tc) * q.ld_c + r0 + l * 8;
        if (nr >= 8) {
          *reinterpret_cast<uint2*>(out) = w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < nr) out[e] = (uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
        }
      }
    }
  }
  if (q.col_partial) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s = __fadd_rn(s, v[i][e]);
      red[g][l * 8 + e] = f2u(s);
    }
    __syncthreads();
    if (threadIdx.x < TILE && c0 + threadIdx.x < q.cols) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < 16; ++w) s = __fadd_rn(s, u2f(red[w][threadIdx.x]));
      q.col_partial[(int64_t)blockIdx.y * q.cols + c0 + threadIdx.x] = s;
    }
  }
}

template <bool BF16, bool E5M2>
void launch(const QArgs& q, const DropSpec& d, bool square, cudaStream_t s) {
  const int64_t nb = (q.cols + TILE - 1) / TILE, mb = (q.rows + TILE - 1) / TILE;
  if (!square && !q.codes_c && !q.col_partial) {
    const int64_t blocks = (q.rows * nb + 15) / 16;
    rows_kernel<BF16, E5M2><<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, s>>>(q, d);
    return;
  }
  const dim3 grid((unsigned)nb, (unsigned)mb);
  if (square) tile_kernel<BF16, E5M2, true><<<grid, 256, 0, s>>>(q, d);
  else tile_kernel<BF16, E5M2, false><<<grid, 256, 0, s>>>(q, d);
}

// Column sums of the slabs' sums, in slab order.
template <bool BF16>
__global__ void col_sum_kernel(void* out, const float* partial, int64_t parts, int64_t cols) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int64_t i = 0; i < parts; ++i) s = __fadd_rn(s, partial[i * cols + c]);
  if (BF16) static_cast<uint16_t*>(out)[c] = (uint16_t)f_to_bf16_rne(s);
  else static_cast<float*>(out)[c] = s;
}

}  // namespace fp8q
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_fp8_quantize(const advopt_fp8_quant_args* a, void* stream) {
  const char* where = "advopt_fp8_quantize: bad arguments";
  if (!a || a->rows < 0 || a->cols < 0 || a->ldx < a->cols) return set_error(ADVOPT_E_INVALID, where);
  if (a->x_dtype != ADVOPT_DT_F32 && a->x_dtype != ADVOPT_DT_BF16)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_quantize: float32 and bfloat16 inputs are supported");
  if ((a->code != ADVOPT_FP8_E4M3 && a->code != ADVOPT_FP8_E5M2) || (a->tile != 0 && a->tile != 1))
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_quantize: unknown code type or block shape");
  if (const char* why = drop_check(a->drop)) return set_error(ADVOPT_E_INVALID, why);
  if (a->rows == 0 || a->cols == 0) return ADVOPT_OK;
  const int64_t nb = (a->cols + 127) / 128, mb = (a->rows + 127) / 128;
  if (!a->x || (!a->codes_r && !a->codes_c) || (a->codes_r && !a->scales_r) || (a->codes_c && !a->scales_c))
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_quantize: null input or output");
  if ((a->codes_r && (a->ld_r < a->cols || a->ld_r % 16 || reinterpret_cast<uintptr_t>(a->codes_r) % 16 || a->ld_sr < nb)) ||
      (a->codes_c && (a->ld_c < a->rows || a->ld_c % 16 || reinterpret_cast<uintptr_t>(a->codes_c) % 16 || a->ld_sc < mb)))
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_quantize: codes must be 16-byte aligned with pitches that hold a row");
  if (nb > 0x7fffffff || mb > 65535) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_quantize: at most 8388480 rows");
  const int64_t es = a->x_dtype == ADVOPT_DT_BF16 ? 2 : 4;
  fp8q::QArgs q;
  q.x = a->x;
  q.ldx = a->ldx;
  q.rows = a->rows;
  q.cols = a->cols;
  q.codes_r = a->codes_r;
  q.ld_r = a->ld_r;
  q.scales_r = a->scales_r;
  q.ld_sr = a->ld_sr;
  q.codes_c = a->codes_c;
  q.ld_c = a->ld_c;
  q.scales_c = a->scales_c;
  q.ld_sc = a->ld_sc;
  q.col_partial = a->col_partial;
  q.vec = reinterpret_cast<uintptr_t>(a->x) % 16 == 0 && (a->ldx * es) % 16 == 0;
  q.drop = a->drop.threshold > 0;
  const DropSpec d = drop_spec(a->drop);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool sq = a->tile != 0;
  if (a->x_dtype == ADVOPT_DT_BF16) {
    if (a->code == ADVOPT_FP8_E5M2) fp8q::launch<true, true>(q, d, sq, s);
    else fp8q::launch<true, false>(q, d, sq, s);
  } else {
    if (a->code == ADVOPT_FP8_E5M2) fp8q::launch<false, true>(q, d, sq, s);
    else fp8q::launch<false, false>(q, d, sq, s);
  }
  return check_cuda(cudaGetLastError(), "advopt_fp8_quantize");
}

extern "C" int advopt_col_sum(void* out, const float* partial, int64_t parts, int64_t cols, int32_t dtype,
                              void* stream) {
  if (parts < 0 || cols < 0 || (cols > 0 && (!out || (parts > 0 && !partial))))
    return set_error(ADVOPT_E_INVALID, "advopt_col_sum: bad arguments");
  if (dtype != ADVOPT_DT_F32 && dtype != ADVOPT_DT_BF16)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_col_sum: float32 and bfloat16 outputs are supported");
  if (cols == 0) return ADVOPT_OK;
  const unsigned grid = (unsigned)((cols + 127) / 128);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == ADVOPT_DT_BF16) fp8q::col_sum_kernel<true><<<grid, 128, 0, s>>>(out, partial, parts, cols);
  else fp8q::col_sum_kernel<false><<<grid, 128, 0, s>>>(out, partial, parts, cols);
  return check_cuda(cudaGetLastError(), "advopt_col_sum");
}
