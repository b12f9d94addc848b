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

constexpr uint32_t INF_BITS = 0x7f800000u;
// |x|'s bits; CAREFUL: 0 for an infinity or NaN (they do not enter a block's scale).
template <bool CAREFUL>
__device__ __forceinline__ uint32_t abs_bits(float x) {
  const uint32_t a = f2u(x) & 0x7fffffffu;
  return CAREFUL && a >= INF_BITS ? 0u : a;
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

// Four codes of a * 2^-e ..; CAREFUL: an infinity becomes NaN (0 * inf), a
// finite product is unchanged (adding 0 of its sign).
template <bool E5M2, bool CAREFUL>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inv) {
  float2 x = mul2(make_float2(a, b), splat2(inv)), y = mul2(make_float2(c, d), splat2(inv));
  if (CAREFUL) {
    x = fma2(make_float2(a, b), splat2(0.0f), x);
    y = fma2(make_float2(c, d), splat2(0.0f), y);
  }
  uint32_t r;
  if (E5M2)
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e5m2x2.f32 l, %2, %1;\n cvt.rn.satfinite.e5m2x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}\n"
        : "=r"(r) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  else
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}\n"
        : "=r"(r) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
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

// Eight consecutive elements of a row.  bf16 ones stay packed: half the
// registers, and their magnitudes are compared two at a time.
struct Row8F {
  float v[8];
  __device__ __forceinline__ float at(int e) const { return v[e]; }
  template <bool CAREFUL>
  __device__ __forceinline__ uint32_t top() const {
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, abs_bits<CAREFUL>(v[e]));
    return a;
  }
};
struct Row8H {
  uint32_t w[4];
  __device__ __forceinline__ float at(int e) const { return u2f((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16); }
  template <bool CAREFUL>
  __device__ __forceinline__ uint32_t top() const {
    if (CAREFUL) {
      uint32_t a = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) a = max(a, abs_bits<true>(at(e)));
      return a;
    }
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu),
                                __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    return max(m << 16, m & 0xFFFF0000u);
  }
};
// bf16 with a dropout: the dropped halves are 0 and the values' common factor
// is applied as they are used, so the elements stay packed (8192 x 4096, both
// layouts: 47 us, as float32 52, without a dropout 26; the Philox rounds are
// most of the rest).  The largest product is the product with the largest
// element, since rounding is monotonic.
struct Row8D : Row8H {
  float f;
  __device__ __forceinline__ float at(int e) const { return __fmul_rn(Row8H::at(e), f); }
  template <bool CAREFUL>
  __device__ __forceinline__ uint32_t top() const {
    if (!CAREFUL) return f2u(__fmul_rn(u2f(Row8H::top<false>()), f));
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, abs_bits<true>(at(e)));
    return a;
  }
};
template <bool BF16>
__device__ __forceinline__ void load_row(Row8F& r, const void* x, int64_t k0, int nv, bool vec) {
  load8<BF16>(x, k0, nv, vec, r.v);
}
template <bool BF16>
__device__ __forceinline__ void load_row(Row8H& r, const void* x, int64_t k0, int nv, bool vec) {
  const uint16_t* p = static_cast<const uint16_t*>(x) + k0;
  if (vec) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[i] = (2 * i < nv ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < nv ? (uint32_t)p[2 * i + 1] << 16 : 0u);
  }
}
// Eight bf16 elements of each of eight rows whose starts are not 16-byte
// aligned (`at`: the lane's first element's address; all lanes take part): a
// lane loads the aligned 16 bytes its elements begin in, takes the next 16
// from the lane behind (the last lane loads them too, where it needs them) and
// shifts: 8192 x 4097 takes 36 us, element by element 50.  float32 rows, whose
// elements are loads of 4 bytes, gain nothing by it (54 us either way).  Every
// aligned 16 bytes that are read hold an element of the row, so
// the reads stay in the matrix's memory to within those 16 bytes.
__device__ __forceinline__ void shifted(const uint4& a, const uint4& b, uint32_t halves, uint32_t (&w)[4]) {
  const bool by4 = halves & 4, by2 = halves & 2, by1 = halves & 1;
  const uint32_t s0 = by4 ? a.z : a.x, s1 = by4 ? a.w : a.y, s2 = by4 ? b.x : a.z, s3 = by4 ? b.y : a.w, s4 = by4 ? b.z : b.x,
                 s5 = by4 ? b.w : b.y;
  const uint32_t t[5] = {by2 ? s1 : s0, by2 ? s2 : s1, by2 ? s3 : s2, by2 ? s4 : s3, by2 ? s5 : s4};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = by1 ? __funnelshift_r(t[i], t[i + 1], 16) : t[i];
}
__device__ __forceinline__ uint4 from_lane_behind(const uint4& a) {
  return make_uint4(__shfl_down_sync(0xffffffffu, a.x, 1, 16), __shfl_down_sync(0xffffffffu, a.y, 1, 16),
                    __shfl_down_sync(0xffffffffu, a.z, 1, 16), __shfl_down_sync(0xffffffffu, a.w, 1, 16));
}
// `at`: the lane's first element's address; all lanes of the warp take part.
__device__ __forceinline__ void load_rows_unaligned(Row8H (&v)[8], const unsigned char* at, int64_t pitch) {
  const bool last = (threadIdx.x & 15) == 15;
  uint4 a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned char* p = at + i * pitch;
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
    const uint4* q = reinterpret_cast<const uint4*>(p - off);
    a[i] = __ldg(q);
    if (last && off) b[i] = __ldg(q + 1);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 n = from_lane_behind(a[i]);
    if (!last) b[i] = n;
    shifted(a[i], b[i], ((uint32_t)reinterpret_cast<uintptr_t>(at + i * pitch) & 15u) >> 1, v[i].w);
  }
}
__device__ __forceinline__ void load_rows_unaligned(Row8D (&v)[8], const unsigned char* at, int64_t pitch) {
  Row8H h[8];
  load_rows_unaligned(h, at, pitch);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i].w[e] = h[i].w[e];
}
__device__ __forceinline__ void load_rows_unaligned(Row8F (&v)[8], const unsigned char* at, int64_t pitch) {
  Row8H h[8];
  load_rows_unaligned(h, at, pitch);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i].v[e] = h[i].at(e);
}
__device__ __forceinline__ void drop_row(Row8F& r, const DropSpec& d, uint32_t step, uint64_t k0) { drop8(r.v, d, step, k0); }
__device__ __forceinline__ void drop_row(Row8H&, const DropSpec&, uint32_t, uint64_t) {}   // Row8D's part
__device__ __forceinline__ void drop_row(Row8D& r, const DropSpec& d, uint32_t step, uint64_t k0) {
  drop_packed(r.w, d, step, k0);
}
__device__ __forceinline__ void set_factor(Row8F&, const DropSpec&) {}
__device__ __forceinline__ void set_factor(Row8H&, const DropSpec&) {}
__device__ __forceinline__ void set_factor(Row8D& r, const DropSpec& d) { r.f = d.scale; }   // one value, of every row

__device__ __forceinline__ void store_codes(uint8_t* out, uint32_t w0, uint32_t w1, int nv) {
  if (nv == 8) {
    *reinterpret_cast<uint2*>(out) = make_uint2(w0, w1);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < nv) out[e] = (uint8_t)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
  }
}

template <bool E5M2, bool CAREFUL, class Row>
__device__ __forceinline__ void code_row(const Row& r, uint32_t byte, uint8_t* out, int nv) {
  const float inv = inv_scale(byte);
  store_codes(out, code4<E5M2, CAREFUL>(r.at(0), r.at(1), r.at(2), r.at(3), inv),
              code4<E5M2, CAREFUL>(r.at(4), r.at(5), r.at(6), r.at(7), inv), nv);
}

// The largest over a half-warp's sixteen lanes.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// ---- rows only, 1 x 128 blocks: sixteen lanes per block, eight elements a lane ----
// For few blocks, which it spreads over all SMs; the tile kernel reads eight
// rows a lane and shares the work of finding their scales.
template <bool BF16, bool E5M2, class Row>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ QArgs q, const __grid_constant__ DropSpec d) {
  // a product behind this kernel may set itself up meanwhile; it waits for the codes
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t step = q.drop ? drop_step(d) : 0u;
  const int l16 = threadIdx.x & 15;
  const int64_t nb = (q.cols + TILE - 1) / TILE;
  const int64_t units = q.rows * nb;
  const int64_t stride = (int64_t)gridDim.x * (blockDim.x / 16);
  // a half-warp's block and how far the next one is: two divisions in all, not one a block
  const int64_t u0 = (int64_t)blockIdx.x * (blockDim.x / 16) + (threadIdx.x >> 4);
  int64_t r = u0 / nb, b = u0 - r * nb;
  const int64_t dr = stride / nb, db = stride - dr * nb;
  // both halves of a warp take every trip: the votes below name all lanes
  for (int64_t u = u0; (u & ~(int64_t)1) < units; u += stride) {
    const bool live = u < units;
    const int64_t c0 = b * TILE + l16 * 8;
    const int nv = !live || c0 >= q.cols ? 0 : q.cols - c0 < 8 ? (int)(q.cols - c0) : 8;
    Row v;
    load_row<BF16>(v, q.x, r * q.ldx + c0, nv, q.vec && nv == 8);
    set_factor(v, d);
    if (q.drop && nv) drop_row(v, d, step, (uint64_t)(r * q.cols + c0));
    uint32_t a = half_warp_max(v.template top<false>());
    uint8_t* out = q.codes_r + r * q.ld_r + c0;
    if (!__any_sync(0xffffffffu, a >= INF_BITS)) {
      a = scale_byte<E5M2>(a);
      if (nv) code_row<E5M2, false>(v, a, out, nv);
    } else {
      a = scale_byte<E5M2>(half_warp_max(v.template top<true>()));
      if (nv) code_row<E5M2, true>(v, a, out, nv);
    }
    if (live && l16 == 0) q.scales_r[r * q.ld_sr + b] = (uint8_t)a;
    r += dr;
    b += db;
    if (b >= nb) {
      b -= nb;
      ++r;
    }
  }
}

// ---- one 128 x 128 tile per CTA: any layout, both block shapes, column sums ----
// Thread (g, l) of 16 x 16 holds rows 8g .. 8g+7, columns 8l .. 8l+7.
struct TileShared {
  uint32_t red[8][TILE];     // column maxima of a warp's 16 rows; column sums
  uint8_t turned[TILE * TILE];
  uint32_t col_byte[TILE];
  uint32_t warp_top[8];
};

// Columns' maxima over a warp's 16 rows, into red[warp].
template <bool CAREFUL, class Row>
__device__ __forceinline__ void column_tops_each(const Row (&v)[8], TileShared& s) {
  const int warp = threadIdx.x >> 5, l = threadIdx.x & 15;
  uint32_t a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a[e] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[e] = max(a[e], abs_bits<CAREFUL>(v[i].at(e)));
    a[e] = max(a[e], __shfl_xor_sync(0xffffffffu, a[e], 16));
  }
  if ((threadIdx.x & 16) == 0) {
    *reinterpret_cast<uint4*>(&s.red[warp][l * 8]) = make_uint4(a[0], a[1], a[2], a[3]);
    *reinterpret_cast<uint4*>(&s.red[warp][l * 8 + 4]) = make_uint4(a[4], a[5], a[6], a[7]);
  }
}
template <class Row>
__device__ __forceinline__ void column_tops_packed(const Row (&v)[8], float f, TileShared& s) {
  const int warp = threadIdx.x >> 5, l = threadIdx.x & 15;
  uint32_t a[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = __vmaxu2(m, v[i].w[j] & 0x7FFF7FFFu);
    }
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 16));
    a[2 * j] = f2u(__fmul_rn(u2f(m << 16), f));
    a[2 * j + 1] = f2u(__fmul_rn(u2f(m & 0xFFFF0000u), f));
  }
  if ((threadIdx.x & 16) == 0) {
    *reinterpret_cast<uint4*>(&s.red[warp][l * 8]) = make_uint4(a[0], a[1], a[2], a[3]);
    *reinterpret_cast<uint4*>(&s.red[warp][l * 8 + 4]) = make_uint4(a[4], a[5], a[6], a[7]);
  }
}
template <bool CAREFUL>
__device__ __forceinline__ void column_tops(const Row8F (&v)[8], TileShared& s) {
  column_tops_each<CAREFUL>(v, s);
}
template <bool CAREFUL>
__device__ __forceinline__ void column_tops(const Row8H (&v)[8], TileShared& s) {
  if (CAREFUL) column_tops_each<true>(v, s);
  else column_tops_packed(v, 1.0f, s);
}
template <bool CAREFUL>
__device__ __forceinline__ void column_tops(const Row8D (&v)[8], TileShared& s) {
  if (CAREFUL) column_tops_each<true>(v, s);
  else column_tops_packed(v, v[0].f, s);
}

// The largest of each of eight rows over a half-warp: lane l gets row l & 7's.
// Halving what is exchanged at each step takes 8 shuffles; every row by itself
// takes 32, and each lane would work out all eight scales.
__device__ __forceinline__ uint32_t scatter_max(const uint32_t (&a)[8]) {
  const bool l0 = threadIdx.x & 1, l1 = threadIdx.x & 2, l2 = threadIdx.x & 4;
  uint32_t b[4], c[2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = max(l0 ? a[2 * i + 1] : a[2 * i], __shfl_xor_sync(0xffffffffu, l0 ? a[2 * i] : a[2 * i + 1], 1));
#pragma unroll
  for (int i = 0; i < 2; ++i)
    c[i] = max(l1 ? b[2 * i + 1] : b[2 * i], __shfl_xor_sync(0xffffffffu, l1 ? b[2 * i] : b[2 * i + 1], 2));
  const uint32_t d = max(l2 ? c[1] : c[0], __shfl_xor_sync(0xffffffffu, l2 ? c[0] : c[1], 4));
  return max(d, __shfl_xor_sync(0xffffffffu, d, 8));
}

// FULL: the tile lies inside the matrix.
template <bool E5M2, bool SQUARE, bool CAREFUL, bool FULL, class Row>
__device__ __forceinline__ void tile_body(const QArgs& q, const Row (&v)[8], TileShared& s, int64_t tr, int64_t tc, int nv) {
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t r0 = tr * TILE, c0 = tc * TILE;
  const int64_t c = c0 + l * 8;
  uint32_t square_byte = 0;
  if (SQUARE) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, v[i].template top<CAREFUL>());
    a = __reduce_max_sync(0xffffffffu, a);
    if ((threadIdx.x & 31) == 0) s.warp_top[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) a = max(a, s.warp_top[w]);
    square_byte = scale_byte<E5M2>(a);
    if (threadIdx.x == 0) {
      if (q.codes_r) q.scales_r[tr * q.ld_sr + tc] = (uint8_t)square_byte;
      if (q.codes_c) q.scales_c[tc * q.ld_sc + tr] = (uint8_t)square_byte;
    }
  }
  if (!SQUARE && q.codes_c) column_tops<CAREFUL>(v, s);
  if (q.codes_r) {
    uint32_t row_byte = square_byte;   // of row 8g + (l & 7)
    if (!SQUARE) {
      uint32_t a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = v[i].template top<CAREFUL>();
      row_byte = scale_byte<E5M2>(scatter_max(a));
      if (l < 8 && (FULL || r0 + g * 8 + l < q.rows)) q.scales_r[(r0 + g * 8 + l) * q.ld_sr + tc] = (uint8_t)row_byte;
    }
    uint8_t* out = q.codes_r + (r0 + g * 8) * q.ld_r + c;
    const int left = FULL ? 8 : q.rows - r0 - g * 8 < 8 ? (int)(q.rows - r0 - g * 8) : 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t sb = SQUARE ? square_byte : __shfl_sync(0xffffffffu, row_byte, i, 16);
      if (FULL || (i < left && nv)) code_row<E5M2, CAREFUL>(v[i], sb, out, FULL ? 8 : nv);
      out += q.ld_r;
    }
  }
  if (q.codes_c) {
    if (!SQUARE) {
      __syncthreads();
      if (threadIdx.x < TILE) {
        uint32_t a = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) a = max(a, s.red[w][threadIdx.x]);
        const uint32_t sb = scale_byte<E5M2>(a);
        s.col_byte[threadIdx.x] = sb;
        if (c0 + threadIdx.x < q.cols) q.scales_c[(c0 + threadIdx.x) * q.ld_sc + tr] = (uint8_t)sb;
      }
      __syncthreads();
    }
    // column 8l + e of the tile is row 8l + e of `turned`: 16 chunks of 8
    // bytes, chunk g kept at g ^ l so that a half-warp's stores (one chunk
    // each of 16 rows) and its loads (one row's 16 chunks) touch all banks
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float inv = inv_scale(SQUARE ? square_byte : s.col_byte[l * 8 + e]);
      const uint32_t w0 = code4<E5M2, CAREFUL>(v[0].at(e), v[1].at(e), v[2].at(e), v[3].at(e), inv);
      const uint32_t w1 = code4<E5M2, CAREFUL>(v[4].at(e), v[5].at(e), v[6].at(e), v[7].at(e), inv);
      *reinterpret_cast<uint2*>(s.turned + (l * 8 + e) * TILE + ((g ^ l) << 3)) = make_uint2(w0, w1);
    }
    __syncthreads();
    const int64_t rows_left = q.rows - r0 - l * 8;   // rows of x from this thread's chunk on
    const int nr = FULL || rows_left >= 8 ? 8 : rows_left > 0 ? (int)rows_left : 0;
    uint8_t* out = q.codes_c + (c0 + g) * q.ld_c + r0 + l * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = i * 16 + g;
      if (FULL || (c0 + col < q.cols && nr > 0)) {
        const uint2 w = *reinterpret_cast<const uint2*>(s.turned + col * TILE + ((l ^ (col >> 3)) << 3));
        store_codes(out, w.x, w.y, FULL ? 8 : nr);
      }
      out += 16 * q.ld_c;
    }
  }
}

// Packed bf16 rows take 80 registers and three CTAs an SM, which spills up to 84
// bytes a thread; with two CTAs of 128 registers nothing spills and 8192 x 4096
// in both layouts takes 30.0 us instead of 25.8 (2048 x 2048, 256 tiles: 4.5,
// 4.8).  float32 rows have room for two: 35.8 us, 0.86 of HBM.
template <bool BF16, bool E5M2, bool SQUARE, class Row>
__global__ void __launch_bounds__(256, sizeof(Row) == 16 ? 3 : 2) tile_kernel(const __grid_constant__ QArgs q, const __grid_constant__ DropSpec d) {
  __shared__ __align__(16) TileShared s;
  // a product behind this kernel may set itself up meanwhile; it waits for the codes
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t step = q.drop ? drop_step(d) : 0u;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const uint32_t across = (uint32_t)((q.cols + TILE - 1) / TILE);
  const int64_t tr = blockIdx.x / across, tc = blockIdx.x - (uint32_t)tr * across;
  const int64_t r0 = tr * TILE, c0 = tc * TILE;
  const int64_t c = c0 + l * 8;
  const int nv = c >= q.cols ? 0 : q.cols - c < 8 ? (int)(q.cols - c) : 8;
  const bool full = r0 + TILE <= q.rows && c0 + TILE <= q.cols;
  Row v[8];
  int64_t at = (r0 + g * 8) * q.ldx + c;
  if (BF16 && full && !q.vec) {
    load_rows_unaligned(v, static_cast<const unsigned char*>(q.x) + at * 2, q.ldx * 2);
  } else if (full && q.vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i, at += q.ldx) load_row<BF16>(v[i], q.x, at, 8, true);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i, at += q.ldx) {
      const int n = r0 + g * 8 + i < q.rows ? nv : 0;
      load_row<BF16>(v[i], q.x, at, n, q.vec && n == 8);
    }
  }
  if (q.drop) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + g * 8 + i;
      set_factor(v[i], d);
      if (r < q.rows && nv) drop_row(v[i], d, step, (uint64_t)(r * q.cols + c));
    }
  }
  if (q.col_partial) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) t[e] = __fadd_rn(t[e], v[i].at(e));
      t[e] = __fadd_rn(t[e], __shfl_xor_sync(0xffffffffu, t[e], 16));
    }
    if ((threadIdx.x & 16) == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s.red[threadIdx.x >> 5][l * 8 + e] = f2u(t[e]);
    }
    __syncthreads();
    if (threadIdx.x < TILE && c0 + threadIdx.x < q.cols) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t = __fadd_rn(t, u2f(s.red[w][threadIdx.x]));
      q.col_partial[tr * q.cols + c0 + threadIdx.x] = t;
    }
  }
  // infinities and NaN are looked for once, and only a tile that has some pays for them
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, v[i].template top<false>());
  if (__syncthreads_or(a >= INF_BITS)) tile_body<E5M2, SQUARE, true, false>(q, v, s, tr, tc, nv);
  else if (full) tile_body<E5M2, SQUARE, false, true>(q, v, s, tr, tc, nv);
  else tile_body<E5M2, SQUARE, false, false>(q, v, s, tr, tc, nv);
}

template <bool BF16, bool E5M2, class Row>
void launch_row(const QArgs& q, const DropSpec& d, bool square, cudaStream_t s) {
  const int64_t nb = (q.cols + TILE - 1) / TILE, mb = (q.rows + TILE - 1) / TILE;
  if (!square && !q.codes_c && !q.col_partial) {
    const int64_t blocks = (q.rows * nb + 15) / 16;
    // 7 x 4096 bf16: 1.7 us, 2.7 in tiles; 1000 x 2048 f32: 4.0 us, 2.9 in tiles
    if (blocks < 148 * 2) {
      rows_kernel<BF16, E5M2, Row><<<(unsigned)blocks, 256, 0, s>>>(q, d);
      return;
    }
  }
  const unsigned grid = (unsigned)(nb * mb);
  if (square) tile_kernel<BF16, E5M2, true, Row><<<grid, 256, 0, s>>>(q, d);
  else tile_kernel<BF16, E5M2, false, Row><<<grid, 256, 0, s>>>(q, d);
}

template <bool BF16, bool E5M2>
void launch(const QArgs& q, const DropSpec& d, bool square, cudaStream_t s) {
  if (!BF16) launch_row<BF16, E5M2, Row8F>(q, d, square, s);
  else if (q.drop) launch_row<BF16, E5M2, Row8D>(q, d, square, s);
  else launch_row<BF16, E5M2, Row8H>(q, d, square, s);
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
  if (nb > 0x7fffffff || mb > 0x7fffffff / nb)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_quantize: at most 2^31 - 1 tiles of 128 x 128");
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
