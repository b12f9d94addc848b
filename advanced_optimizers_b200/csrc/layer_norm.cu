// Layer norm: y = (x - mean) * rstd * w + b over rows, and its gradients
//   g = dy * w, h = (x - mean) * rstd,
//   dx = rstd * (g - mean of g - h * mean of g h), dw = sum of dy h, db = sum of dy.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and
// writes dx, each once (16384 x 4096 bf16: 45 and 76 us for 41 and 61 of HBM's;
// the second is bound by its instructions at 16 warps an SM, 26 an element).
// A row stays in the registers of one warp (up to 1024 columns; bf16 backward
// 768), one CTA (up to 16384 forward, 8192 backward) or a cluster of up to eight
// (up to 65536), so the variance is that of the differences from the mean, in
// float32, without a second read; h is rstd times these differences.  Wider rows
// are read again (from L2).  dw and db are summed down the columns that a thread
// holds, over all rows its CTA takes (of the widest rows by a kernel of their own
// that reads again); the CTAs' sums are added in order by one more launch, so
// that results repeat bit for bit.
#include <cooperative_groups.h>

#include <atomic>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace cg = cooperative_groups;

namespace advopt {
namespace ln {

constexpr int WARPS = 8;      // rows at a time of a CTA whose warps take a row each
constexpr int PAYLOAD = 30;   // lanes of a warp whose vectors are its own, of unaligned rows

// Sums of N values (1, 2 or 4) over the warp: lane l gets value l / (32 / N).
// Two values are halved with one exchange, so that N cost little more than one.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  float a = v[0];
  int o = 16;
  if constexpr (N == 2) {
    a = __fadd_rn(lane & 16 ? v[1] : v[0], __shfl_xor_sync(0xffffffffu, lane & 16 ? v[0] : v[1], 16));
    o = 8;
  }
  if constexpr (N == 4) {
    float h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = __fadd_rn(lane & 16 ? v[2 + i] : v[i], __shfl_xor_sync(0xffffffffu, lane & 16 ? v[i] : v[2 + i], 16));
    a = __fadd_rn(lane & 8 ? h[1] : h[0], __shfl_xor_sync(0xffffffffu, lane & 8 ? h[0] : h[1], 8));
    o = 4;
  }
#pragma unroll
  for (; o > 0; o >>= 1) a = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// Sums of N values over the warp (Q = 0) or the CTA of up to 4 Q warps; every
// thread gets them.  `red` has room for two rounds, so that one barrier a round
// is enough; what it holds for warps that are not there is 0 (clear_sums).
template <int N, int Q>
__device__ __forceinline__ void row_sum(float (&v)[N], float4 (*red)[Q ? Q * N : 1], int& round) {
  const float a = warp_sums<N>(v);
  if constexpr (Q == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = N == 1 ? a : __shfl_sync(0xffffffffu, a, i * (32 / N));
  } else {
    float4* r = red[round];
    round ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane % (32 / N) == 0) reinterpret_cast<float*>(r + lane / (32 / N) * Q)[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const float4 q = r[i * Q + k];
        s = add2(s, add2(make_float2(q.x, q.y), make_float2(q.z, q.w)));
      }
      v[i] = __fadd_rn(s.x, s.y);
    }
  }
}
template <int N, int Q>
__device__ __forceinline__ void clear_sums(float4 (*red)[Q ? Q * N : 1]) {
  if constexpr (Q > 0) {
    for (int i = threadIdx.x; i < 2 * Q * N; i += blockDim.x) red[i / (Q * N)][i % (Q * N)] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
  }
}
// A row's mean from its sum and 1 / cols: the product, and what is left of the sum (exact in one fma) once more, so that the mean is exact where
// it is a float.
__device__ __forceinline__ float mean_of(float sum, float cols, float inv) {
  const float m = __fmul_rn(sum, inv);
  return __fmaf_rn(__fmaf_rn(-m, cols, sum), inv, m);
}
// A CTA's place in a cluster of up to 8 that share a row (1 without one), and the row's sums over them.  Timed against two
// reads of a row and a third for dw and db, backward: 4096 x 16384 bf16 150 -> 117 us, 8192 x 12288 230 -> 168, 2048 x
// 16384 float32 169 -> 84, 4000 x 12005 float32 492 -> 143; forward, beyond 16384 columns, against three reads: 1024 x
// 32768 float32 86 -> 70, 1000 x 40001 bf16 172 -> 76.
constexpr int MOST_CTAS = 8;
template <bool CLUSTER, int N>
struct Team {
  uint32_t ctas, rank;
  __device__ __forceinline__ Team() : ctas(1), rank(0) {
    if constexpr (CLUSTER) {
      ctas = cg::this_cluster().num_blocks();
      rank = cg::this_cluster().block_rank();
    }
  }
  // Of the CTA's sums v, which all its threads hold; added in the CTAs' order.  `all` has room for two rounds: a CTA writes
  // a round's place again only after a barrier that the others reach when they have read it.
  __device__ __forceinline__ void sum(float (&v)[N], float (*all)[MOST_CTAS][N], int& round) const {
    if constexpr (CLUSTER) {
      cg::cluster_group cluster = cg::this_cluster();
      float (*p)[N] = all[round];
      round ^= 1;
      if (threadIdx.x < ctas) {
        float* to = cluster.map_shared_rank(p[rank], threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = v[i];
      }
      cluster.sync();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[0][i];
      for (uint32_t k = 1; k < ctas; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], p[k][i]);
    }
  }
};
// Q of a kernel for rows of up to `threads` threads (32: a warp's).
__host__ __device__ constexpr int quads(int threads) { return threads == 32 ? 0 : (threads + 127) / 128; }

// How rows lie.  ALIGNED: all on 16-byte boundaries.  PHASE: all of a pass's
// tensors lie the same way, and a thread's rows are eight apart, so that they
// all begin at the same place between two boundaries; it takes the 16 bytes
// between boundaries as they are, with the columns that these hold.  SHIFT:
// anything else; what is read is shifted into place, and so is what is written.
// Timed, PHASE against SHIFT: 10000 x 5003 bf16 47 us forward for 73 and 91
// backward for 100, float32 69 for 100 and 107 for 154, 16384 x 999 float32 24
// for 44 and 38 for 81; aligned rows of 5000 take 40 and 67 in bf16.
constexpr int ALIGNED = 0, PHASE = 1, SHIFT = 2;

// A thread's columns: NV vectors of 16 bytes of x, each warp's (or CTA's) next
// to one another.  PHASE: `k` elements ahead of the row share its first 16
// bytes.  SHIFT: a warp's first lane repeats the vector ahead of the warp's,
// whose last elements the next lane stores, and its last lane the one behind,
// whose first ones the lane before reads; they are in no sum.
template <bool BF16, int NV, int MODE>
struct Columns {
  static constexpr int E = BF16 ? 8 : 4;
  static constexpr uint32_t WHOLE = (1u << E) - 1;
  static_assert(NV * E <= 32, "a bit for each element");
  int first, each;                                  // vector v begins at first + v * each
  uint32_t row, mine;                               // a bit for each element: of the row, and to be summed by this thread
  uint32_t ragged;                                  // a bit for each vector: the row begins or ends within one of the warp's
  __device__ __forceinline__ int c(int v) const { return first + v * each; }
  __device__ __forceinline__ uint32_t bits(int v) const { return row >> (v * E) & WHOLE; }
  __device__ __forceinline__ bool whole(int v) const { return (mine >> (v * E) & WHOLE) == WHOLE; }
  __device__ __forceinline__ bool some(int v) const { return (mine >> (v * E) & WHOLE) != 0; }
  // The same, for a branch in the loop over rows: volatile, since what follows from the bits would be worked out ahead of
  // the loop and take more registers than there are.
  __device__ __forceinline__ static uint32_t here(uint32_t bits) {
    uint32_t b;
    asm volatile("mov.b32 %0, %1;" : "=r"(b) : "r"(bits));
    return b;
  }
  __device__ __forceinline__ void init(int cols, bool warp_rows, int rank, int k) {
    const int lane = threadIdx.x & 31, warp = warp_rows ? 0 : threadIdx.x >> 5, warps = warp_rows ? 1 : blockDim.x >> 5;
    constexpr int LANES = MODE == SHIFT ? PAYLOAD : 32;
    first = ((rank * NV * warps + warp) * LANES + lane - (MODE == SHIFT ? 1 : 0)) * E - (MODE == PHASE ? k : 0);
    each = warps * LANES * E;
    row = ragged = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      uint32_t q = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) q |= c(v) + e >= 0 && c(v) + e < cols ? 1u << e : 0u;
      if (MODE != ALIGNED && __any_sync(0xffffffffu, q && q != WHOLE)) ragged |= 1u << v;
      row |= q << (v * E);
    }
    mine = MODE == SHIFT && (lane == 0 || lane > PAYLOAD) ? 0u : row;
  }
  // Zeros in those of vectors v (N of them) that are outside the row, where the row begins or ends in one of the warp's.
  template <class X, int N>
  __device__ __forceinline__ void clear(int v, X* const (&x)[N]) const {
    if (MODE == ALIGNED || !(ragged >> v & 1u)) return;
    const uint32_t bits = here(row) >> (v * E);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = BF16 ? (bits >> (2 * i) & 1u ? 0xFFFFu : 0u) | (bits >> (2 * i + 1) & 1u ? 0xFFFF0000u : 0u) : bits >> i & 1u ? 0xFFFFFFFFu : 0u;
#pragma unroll
      for (int n = 0; n < N; ++n) x[n]->w[i] &= m;
    }
  }
};

// Words k .. k + 4 of eight, shifted by `bits` (0 or 16): 16 bytes from byte 4 k + bits / 8 on.  k and bits are the warp's.
__device__ __forceinline__ void cut(const uint32_t (&t)[8], uint32_t k, uint32_t bits, uint32_t (&w)[4]) {
  const auto from = [&](auto at) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(t[at.value + i], t[at.value + i + 1], bits);
  };
  if (k < 2) {
    if (k == 0) from(std::integral_constant<int, 0>());
    else from(std::integral_constant<int, 1>());
  } else {
    if (k == 2) from(std::integral_constant<int, 2>());
    else from(std::integral_constant<int, 3>());
  }
}

// E elements: those of x's 16 bytes, or the weights that belong to them.
template <bool BF16, int E>
struct Vals {
  static constexpr int W = BF16 ? E / 2 : E;
  uint32_t w[W];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (BF16) return u2f((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
    else return u2f(w[e]);
  }
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(at(2 * i), at(2 * i + 1)); }
  __device__ __forceinline__ void set_pair(int i, float2 v) {   // of float32
    w[2 * i] = f2u(v.x);
    w[2 * i + 1] = f2u(v.y);
  }
  __device__ __forceinline__ void set(const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (BF16) w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
      else w[i] = f2u(v[i]);
    }
  }
  // `absent` where there are no weights; zeros outside the row; vec: 8-byte aligned
  __device__ __forceinline__ void weights(const void* p, float absent, int c, uint32_t bits, bool vec) {
    if (!p) {
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = absent;
      set(v);
      return;
    }
    if (vec && bits == (1u << E) - 1) {
      const uint2* q = reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(p) + (int64_t)c * (BF16 ? 2 : 4));
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        const uint2 u = __ldg(q + i);
        w[2 * i] = u.x;
        w[2 * i + 1] = u.y;
      }
      return;
    }
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      v[e] = !(bits >> e & 1u) ? 0.0f : BF16 ? bf16_to_f(__ldg(static_cast<const uint16_t*>(p) + c + e)) : __ldg(static_cast<const float*>(p) + c + e);
    set(v);
  }
};

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
// A thread copies the 16 bytes that it will read itself, several rows ahead, so
// that only its own copies have to be waited for.  Rows that do not start on a
// 16-byte boundary are copied from the boundary before: each 16 bytes hold an
// element of the row.  SHIFT: a thread's elements then reach into the next
// lane's.
template <bool BF16, int NV, int MODE, int S>
struct Rows {
  static constexpr int E = BF16 ? 8 : 4, SIZE = BF16 ? 2 : 4;
  using X = Vals<BF16, E>;
  uint4* own;                                       // this thread's of stage 0; shared memory is [S][NV][threads]
  const unsigned char* ahead;                       // the next row to be copied
  const unsigned char* now;                         // and to be read (SHIFT)
  int64_t stride;                                   // bytes from a row to the one that follows here
  uint32_t bytes;                                   // of a row
  uint32_t at, each;                                // this thread's first vector, in bytes from the boundary, and from one to the next
  int to, from;                                     // stages
  int behind;                                       // the next lane's slot; the last lane, which needs none, takes its own

  // 16-byte slots of a CTA
  __host__ __device__ static constexpr int slots_of(int threads) { return S * NV * threads; }
  __device__ __forceinline__ void init(uint4* smem, const void* p, int64_t ld, int64_t row, int64_t step, int cols, const Columns<BF16, NV, MODE>& c) {
    own = smem + threadIdx.x;
    ahead = now = static_cast<const unsigned char*>(p) + row * ld * SIZE;
    stride = step * ld * SIZE;
    bytes = (uint32_t)cols * SIZE;
    to = from = 0;
    behind = (threadIdx.x & 31) == 31 ? 0 : 1;
    const uint32_t o = MODE == PHASE ? (uint32_t)reinterpret_cast<uintptr_t>(ahead) & 15u : 0u;
    ahead -= o;                                     // PHASE: from here on the boundary's
    bytes += o;
    at = (uint32_t)(c.first * SIZE) + o;
    each = (uint32_t)(c.each * SIZE);
  }
  __device__ __forceinline__ static void copy(uint4* slot, const unsigned char* p) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot)), "l"(p) : "memory");
  }
  // The next row, if it is there.
  __device__ __forceinline__ void issue(bool there) {
    if (there) {
      const uint32_t o = MODE == SHIFT ? (uint32_t)reinterpret_cast<uintptr_t>(ahead) & 15u : 0u, end = bytes + o;
      const unsigned char* p = ahead - o;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (at + v * each < end) copy(own + (to * NV + v) * (int)blockDim.x, p + (at + v * each));
    }
    ahead += stride;
    to = to == S - 1 ? 0 : to + 1;
  }
  // The next row's elements, anything outside it.  All lanes take part; the copies have been waited for.
  __device__ __forceinline__ void get(X (&x)[NV]) {
    const uint32_t o = MODE == SHIFT ? (uint32_t)reinterpret_cast<uintptr_t>(now) & 15u : 0u;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const uint4* slot = own + (from * NV + v) * (int)blockDim.x;
      const uint4 q = *slot;
      if (MODE == SHIFT) {
        const uint4 n = slot[behind];
        const uint32_t t[8] = {q.x, q.y, q.z, q.w, n.x, n.y, n.z, n.w};
        cut(t, o >> 2, o & 2 ? 16 : 0, x[v].w);
      } else {
        x[v].w[0] = q.x; x[v].w[1] = q.y; x[v].w[2] = q.z; x[v].w[3] = q.w;
      }
    }
    now += stride;
    from = from == S - 1 ? 0 : from + 1;
  }
};
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// A thread's vector v of an output row.  SHIFT: a lane stores the aligned 16
// bytes that its elements begin in, with the lane before's last ones.  Only a
// row's first and last 16 bytes are not whole.  All lanes take part.
template <bool BF16, int NV, int MODE>
__device__ __forceinline__ void put_row(const Vals<BF16, BF16 ? 8 : 4>& x, unsigned char* row, const Columns<BF16, NV, MODE>& col, int v, int cols) {
  constexpr int SIZE = BF16 ? 2 : 4, E = 16 / SIZE;
  unsigned char* p = row + (int64_t)col.c(v) * SIZE;
  if constexpr (MODE == ALIGNED) {
    if (col.some(v)) *reinterpret_cast<uint4*>(p) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
  } else if constexpr (MODE == PHASE) {
    if (col.whole(v)) *reinterpret_cast<uint4*>(p) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
    if ((col.ragged >> v & 1u) && !col.whole(v) && col.some(v)) {
      const uint32_t bits = col.here(col.row) >> (v * E);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (bits >> e & 1u) {
          if (BF16) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(x.w[(e >> 1) & 3] >> (16 * (e & 1)));
          else reinterpret_cast<uint32_t*>(p)[e] = x.w[e & 3];
        }
    }
  } else {
    const uint32_t o = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
    uint32_t t[8], g[4];   // the previous lane's words, then this lane's
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = __shfl_up_sync(0xffffffffu, x.w[i], 1);
      t[4 + i] = x.w[i];
    }
    if (o) {
      const uint32_t back = 16u - o;
      cut(t, back >> 2, back & 2 ? 16 : 0, g);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = x.w[i];
    }
    const int lane = threadIdx.x & 31, first = col.c(v) - (int)o / SIZE;   // of the row's elements in g
    const bool payload = lane > 0 && lane <= PAYLOAD, whole = first >= 0 && first + E <= cols;
    if (payload && whole) *reinterpret_cast<uint4*>(p - o) = make_uint4(g[0], g[1], g[2], g[3]);
    if (__any_sync(0xffffffffu, payload && !whole && first < cols)) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (payload && !whole && first + e >= 0 && first + e < cols) {
          if (BF16) reinterpret_cast<uint16_t*>(p - o)[e] = (uint16_t)(g[(e >> 1) & 3] >> (16 * (e & 1)));
          else reinterpret_cast<uint32_t*>(p - o)[e] = g[e & 3];
        }
    }
  }
}

// The rows of a CTA (a warp, a cluster): from `first` on, `each` apart within a round, `step` from round to round.  PHASE: a CTA's
// all begin at one place, so eight CTAs make a group (fewer where there are fewer rows); SUMS:
// also those of its warps.
template <int MODE, bool WARP, int RI, bool SUMS>
struct Walk {
  int64_t first, each, step;
  __device__ __forceinline__ Walk(uint32_t cta, uint32_t ctas) {
    const int64_t warp = WARP ? threadIdx.x >> 5 : 0;
    if (MODE == PHASE && (SUMS || !WARP)) {
      constexpr int64_t ROWS = (WARP ? WARPS : RI) * 8;
      first = (int64_t)(cta / 8) * ROWS + warp * 8 + cta % 8;
      each = 8;
      step = (ctas < 8 ? 1 : ctas / 8) * ROWS;
    } else {
      constexpr int64_t ROWS = WARP ? WARPS : RI;
      first = (int64_t)cta * ROWS + warp;
      each = 1;
      step = (int64_t)ctas * ROWS;
    }
  }
};

// Stages: rows of a thread on their way, and the one that it reads.  Timed: four forward cost 60 us where three take
// 48 (4096 x 8192 float32), three backward 87 where two take 84 (16384 x 4096 bf16; float32 70 and 72).
constexpr int FWD_STAGES = 3;
__host__ __device__ constexpr int grad_stages(bool bf16) { return bf16 ? 2 : 3; }
// Rows of a CTA that share a round of sums: two of bf16, but one where the fewer registers let two CTAs run on an SM: 320
// threads and 384 of aligned rows (10000 x 5000: 86 -> 69 us, x 6000: 101 -> 91, and with the statistics read ahead 61 and 75; unaligned ones
// of 320 gained nothing).
__host__ __device__ constexpr bool two_ctas(bool bf16, int max_threads, int mode) { return bf16 && mode == ALIGNED && (max_threads == 320 || max_threads == 384); }
__host__ __device__ constexpr int grad_rows(bool bf16, int max_threads, int mode) {
  return bf16 && max_threads > 32 && !two_ctas(bf16, max_threads, mode) ? 2 : 1;
}

template <bool BX, bool BW, int NV, int MAX_THREADS, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(MAX_THREADS == 32 ? 256 : MAX_THREADS, MAX_THREADS == 32 || MAX_THREADS == 1024 ? 1 : MAX_THREADS == 256 ? (MODE == ALIGNED ? 4 : 3) : 2)
    forward_kernel(const __grid_constant__ advopt_layer_norm_args a, int wvec) {
  constexpr bool WARP = MAX_THREADS == 32;
  constexpr int Q = quads(MAX_THREADS);
  extern __shared__ uint4 smem[];
  __shared__ float4 red[2][Q ? Q : 1];
  const int lane = WARP ? threadIdx.x & 31 : threadIdx.x, cols = (int)a.cols;
  constexpr int S = FWD_STAGES, E = BX ? 8 : 4, P = E / 2;
  __shared__ float all[2][MOST_CTAS][1];
  const Team<CLUSTER, 1> team;
  const Walk<MODE, WARP, 1, false> walk(blockIdx.x / team.ctas, gridDim.x / team.ctas);
  const int64_t step = walk.step;
  int64_t r = walk.first;
  unsigned char* to = static_cast<unsigned char*>(a.y) + r * cols * (BX ? 2 : 4);
  Columns<BX, NV, MODE> col;
  col.init(cols, WARP, (int)team.rank, (int)(reinterpret_cast<uintptr_t>(to) & 15) / (BX ? 2 : 4));
  Rows<BX, NV, MODE, S> rows;
  rows.init(smem, a.x, a.ldx, r, step, cols, col);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    rows.issue(r + s * step < a.rows);
    commit_copies();
  }
  clear_sums<1, Q>(red);
  if constexpr (CLUSTER) cg::this_cluster().sync();   // all its CTAs are there
  Vals<BW, E> w[NV], b[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    w[v].weights(a.weight, 1.0f, col.c(v), col.bits(v), MODE != PHASE && wvec);
    b[v].weights(a.bias, 0.0f, col.c(v), col.bits(v), MODE != PHASE && wvec);
  }
  const float inv = __fdiv_rn(1.0f, (float)cols);
  int round = 0, team_round = 0;
  for (; r < a.rows; r += step, to += step * cols * (BX ? 2 : 4)) {
    wait_copies<S - 2>();
    if (MODE == SHIFT) __syncwarp();   // the next lane's copies are read too
    float2 x[NV][P];
    {
      Vals<BX, E> raw[NV];
      rows.get(raw);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        Vals<BX, E>* const all[1] = {&raw[v]};
        col.clear(v, all);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < P; ++i) x[v][i] = raw[v].pair(i);
    }
    if (MODE == SHIFT) __syncwarp();
    rows.issue(r + (S - 1) * step < a.rows);   // into the stage that was read a row ago
    commit_copies();
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (col.some(v)) {
#pragma unroll
        for (int i = 0; i < P; ++i) s = add2(s, x[v][i]);
      }
    float t[1] = {__fadd_rn(s.x, s.y)};
    row_sum<1, Q>(t, red, round);
    team.sum(t, all, team_round);
    const float mean = mean_of(t[0], (float)cols, inv);
    s = make_float2(0.0f, 0.0f);
    // x - mean from here on: x rstd - (mean rstd), with the product rounded, is off by another 2^-24 |mean| rstd, where the difference is exact
    // for x near the mean (rows of one value become 0)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < P; ++i) x[v][i] = add2(x[v][i], splat2(-mean));
      if (col.whole(v)) {
#pragma unroll
        for (int i = 0; i < P; ++i) s = fma2(x[v][i], x[v][i], s);
      } else if (MODE != ALIGNED && col.some(v)) {
        const uint32_t bits = col.here(col.mine) >> (v * E);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (bits >> (2 * i) & 1u) s.x = __fmaf_rn(x[v][i].x, x[v][i].x, s.x);
          if (bits >> (2 * i + 1) & 1u) s.y = __fmaf_rn(x[v][i].y, x[v][i].y, s.y);
        }
      }
    }
    t[0] = __fadd_rn(s.x, s.y);
    row_sum<1, Q>(t, red, round);
    team.sum(t, all, team_round);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(t[0], inv, a.eps)));
    const float2 rstd2 = splat2(rstd);
    if (a.stats && lane == 0 && team.rank == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(mean, rstd);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float y[E];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 h = mul2(x[v][i], rstd2), q = fma2(h, w[v].pair(i), b[v].pair(i));
        y[2 * i] = q.x;
        y[2 * i + 1] = q.y;
      }
      Vals<BX, E> o;
      o.set(y);
      put_row<BX, NV, MODE>(o, to, col, v, cols);
    }
  }
}

// Sums over a CTA of 1024 threads.
template <int N>
__device__ __forceinline__ void wide_sum(float (&v)[N], float (*red)[32]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = warp_sum(v[i]);
    if ((threadIdx.x & 31) == 0) red[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(red[i][threadIdx.x & 31]);
  __syncthreads();
}

// Rows that no cluster's registers hold, and many aligned bf16 ones: read three times.
template <bool BX, bool BW>
__global__ void __launch_bounds__(1024) wide_forward_kernel(const __grid_constant__ advopt_layer_norm_args a, int vec, int wvec) {
  __shared__ float red[1][32];
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    float t[1] = {0.0f};
    for (int64_t c = threadIdx.x * 8; c < a.cols; c += 8192) {
      Oct<BX> x;
      x.get(a.x, r * a.ldx + c, a.cols - c < 8 ? (int)(a.cols - c) : 8, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[0] = __fadd_rn(t[0], x.at(e));
    }
    wide_sum<1>(t, red);
    const float mean = mean_of(t[0], (float)a.cols, inv);
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
    wide_sum<1>(t, red);
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
// RI rows of a CTA share a round of sums.
template <bool BX, bool BW, int NV, int MAX_THREADS, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(MAX_THREADS == 32 ? 256 : MAX_THREADS, (MAX_THREADS > 256 && !two_ctas(BX, MAX_THREADS, MODE)) || (MAX_THREADS == 32 && NV > 4) ? 1 : 2)
    grad_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int wvec) {
  constexpr bool WARP = MAX_THREADS == 32;
  constexpr int S = grad_stages(BX), E = BX ? 8 : 4, P = E / 2, RI = grad_rows(BX, MAX_THREADS, MODE), Q = quads(MAX_THREADS);
  extern __shared__ uint4 smem[];
  __shared__ float4 red[2][Q ? Q * 2 * RI : 1];
  const int cols = (int)a.cols;
  using R = Rows<BX, NV, MODE, S>;
  __shared__ float all[2][MOST_CTAS][2 * RI];
  const Team<CLUSTER, 2 * RI> team;
  const Walk<MODE, WARP, RI, true> walk(blockIdx.x / team.ctas, gridDim.x / team.ctas);
  const int64_t step = walk.step, each = walk.each;
  int64_t r = walk.first;
  Columns<BX, NV, MODE> col;
  col.init(cols, WARP, (int)team.rank, (int)((reinterpret_cast<uintptr_t>(a.x) + r * a.ldx * (BX ? 2 : 4)) & 15) / (BX ? 2 : 4));
  R xs[RI], dys[RI];
#pragma unroll
  for (int q = 0; q < RI; ++q) {
    xs[q].init(smem + 2 * q * R::slots_of(blockDim.x), a.x, a.ldx, r + q * each, step, cols, col);
    dys[q].init(smem + (2 * q + 1) * R::slots_of(blockDim.x), a.dy, a.lddy, r + q * each, step, cols, col);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      const bool there = r + s * step + q * each < a.rows;
      xs[q].issue(there);
      dys[q].issue(there);
    }
    commit_copies();
  }
  clear_sums<2 * RI, Q>(red);
  if constexpr (CLUSTER) cg::this_cluster().sync();   // all its CTAs are there
  Vals<BW, E> w[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) w[v].weights(a.weight, 1.0f, col.c(v), col.bits(v), MODE != PHASE && wvec);
  float2 dw[NV][P], db[NV][P];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < P; ++i) dw[v][i] = db[v][i] = make_float2(0.0f, 0.0f);
  const float inv = __fdiv_rn(1.0f, (float)cols);
  const int64_t row_bytes = (int64_t)cols * (BX ? 2 : 4);
  unsigned char* to = static_cast<unsigned char*>(a.dx) + r * row_bytes;
  int round = 0, team_round = 0;
  // The next row's statistics are on their way too where a round is one row of bf16 or a cluster's.  Timed with and without, bf16: 10000 x 5000 61 and 79 us, x 6000 75 and 90,
  // 65536 x 768 55 and 60; rounds of two rows, which hide one another's, lose by it (16384 x 4096 84 and 76), float32 ones of no cluster now and then (32768 x
  // 700 55 and 50, 4096 x 1021 26 and 32).
  constexpr bool AHEAD = RI == 1 && (BX || CLUSTER);
  float2 next = make_float2(0.0f, 0.0f);
  if (AHEAD && r < a.rows) next = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * r));
  for (; r < a.rows; r += step, to += step * row_bytes) {
    float2 st[RI];
    bool here[RI];
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      here[q] = q == 0 || r + q * each < a.rows;
      if (AHEAD) st[q] = next;
      else if (here[q]) st[q] = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * (r + q * each)));
    }
    if (AHEAD && r + step < a.rows) next = __ldg(reinterpret_cast<const float2*>(a.stats + 2 * (r + step)));
    wait_copies<S - 2>();
    if (MODE == SHIFT) __syncwarp();   // the next lane's copies are read too
    Vals<BX, E> x[RI][NV], dy[RI][NV];
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      xs[q].get(x[q]);
      dys[q].get(dy[q]);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Vals<BX, E>* const all[4] = {&x[0][v], &dy[0][v], &x[RI - 1][v], &dy[RI - 1][v]};   // of one row: the same twice
      col.clear(v, all);
    }
    if (MODE == SHIFT) __syncwarp();
    // into the stage that was read a round ago
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      const bool there = r + (S - 1) * step + q * each < a.rows;
      xs[q].issue(there);
      dys[q].issue(there);
    }
    commit_copies();
    float t[2 * RI];
    float2 rstd2[RI];
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
      const float mean = st[q].x, rstd = st[q].y;
      rstd2[q] = splat2(rstd);
      if constexpr (!BX) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < P; ++i) x[q][v].set_pair(i, add2(x[q][v].pair(i), splat2(-mean)));   // also what the next lane stores
      }
      if (here[q]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (col.some(v)) {   // x and dy are 0 where a vector is outside its row; h is not a number there only where all of a row's are
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 xm = BX ? add2(x[q][v].pair(i), splat2(-mean)) : x[q][v].pair(i), h = mul2(xm, rstd2[q]), d = dy[q][v].pair(i), g = mul2(d, w[v].pair(i));
              s1 = add2(s1, g);
              s2 = fma2(g, h, s2);
              dw[v][i] = fma2(d, h, dw[v][i]);
              db[v][i] = add2(db[v][i], d);
            }
          }
        }
      }
      t[2 * q] = __fadd_rn(s1.x, s1.y);
      t[2 * q + 1] = __fadd_rn(s2.x, s2.y);
    }
    if (!a.dx) continue;
    row_sum<2 * RI, Q>(t, red, round);
    team.sum(t, all, team_round);
#pragma unroll
    for (int q = 0; q < RI; ++q) {
      if (!here[q]) continue;
      // dx = rstd (g - m1 - m2 rstd (x - mean)); the square of rstd, which may be beyond float32, appears nowhere.  float32 rows have kept x - mean; of
      // bf16 ones, which would take registers for it, slope times the mean is rounded with the rest: their spread is at least 2^-8 /
      // sqrt(cols) of their mean, or nothing (and m2 is 0 with h), so that this is off by 2^-15 of rstd g at most.
      const float mean = st[q].x, rstd = st[q].y, m1 = __fmul_rn(t[2 * q], inv), m2 = __fmul_rn(t[2 * q + 1], inv);
      const float slope = -__fmul_rn(rstd, m2);
      const float2 slope2 = splat2(slope), rest2 = splat2(-__fmul_rn(rstd, BX ? __fmaf_rn(slope, mean, m1) : m1));
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float o[E];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 g = mul2(dy[q][v].pair(i), w[v].pair(i)), p = fma2(fma2(x[q][v].pair(i), slope2, g), rstd2[q], rest2);
          o[2 * i] = p.x;
          o[2 * i + 1] = p.y;
        }
        Vals<BX, E> out;
        out.set(o);
        put_row<BX, NV, MODE>(out, to + q * each * row_bytes, col, v, cols);
      }
    }
  }
  if (!a.work) return;
  float* part = static_cast<float*>(a.work) + (int64_t)(blockIdx.x / team.ctas) * 2 * a.cols;
  if constexpr (WARP) {
    // the warps' sums through shared memory, all of the same columns: [WARPS][2][NV * P][32], added in the warps' order
    wait_copies<0>();
    __syncthreads();
    constexpr int ALL = 2 * NV * P;
    static_assert(WARPS * ALL * 32 * 8 <= 2 * R::slots_of(WARPS * 32) * 16, "the rows' shared memory");
    float2* sh = reinterpret_cast<float2*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        sh[(warp * ALL + v * P + i) * 32 + lane] = dw[v][i];
        sh[(warp * ALL + NV * P + v * P + i) * 32 + lane] = db[v][i];
      }
    __syncthreads();
    for (int j = warp; j < ALL; j += WARPS) {
      float2 t = sh[j * 32 + lane];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) t = add2(t, sh[(k * ALL + j) * 32 + lane]);
      const int m = j % (NV * P), c = col.first + m / P * col.each + m % P * 2;
      float* p = part + j / (NV * P) * cols + c;
      if (MODE == SHIFT && (lane == 0 || lane > PAYLOAD)) continue;
      if (c >= 0 && c < cols) p[0] = t.x;
      if (c + 1 >= 0 && c + 1 < cols) p[1] = t.y;
    }
  } else {
    // in the columns' order through shared memory, so that whole sectors are written; two words in 34 are left free against bank conflicts
    // (1000 x 5003 bf16: 12 us where each thread's own stores took 16)
    wait_copies<0>();
    float* sh = reinterpret_cast<float*>(smem);
    const auto place = [](int i) { return i + (i >> 5) * 2; };
    constexpr int LANES = MODE == SHIFT ? PAYLOAD : 32;
    const int lane31 = threadIdx.x & 31, span = NV * (int)(blockDim.x >> 5) * LANES * E;
    const int begin = col.first - ((int)(threadIdx.x >> 5) * LANES + lane31 - (MODE == SHIFT ? 1 : 0)) * E;   // the CTA's first column
    static_assert(NV * E * 4 * 17 / 16 <= 2 * RI * S * NV * 16, "the rows' shared memory");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
      if (MODE != SHIFT || (lane31 > 0 && lane31 <= PAYLOAD)) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < P; ++i) *reinterpret_cast<float2*>(sh + place(col.c(v) - begin + 2 * i)) = k ? db[v][i] : dw[v][i];
      }
      __syncthreads();
      for (int j = threadIdx.x; j < span; j += blockDim.x)
        if (begin + j >= 0 && begin + j < cols) part[k * cols + begin + j] = sh[place(j)];
    }
  }
}

// Rows that no cluster's registers hold: dx from two reads of a row.
template <bool BX, bool BW>
__global__ void __launch_bounds__(1024) wide_dx_kernel(const __grid_constant__ advopt_layer_norm_grad_args a, int vec, int wvec) {
  __shared__ float red[2][32];
  const float inv = __fdiv_rn(1.0f, (float)a.cols);
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
    wide_sum<2>(t, red);
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
constexpr int64_t SMS = 148;

// Vectors per thread, and threads and CTAs of a row: a warp's where it holds
// the row in `one` to `most` * `one` vectors a lane, else a CTA's of up to
// `threads` with `one` * 2, else those of a cluster: of up to 256 threads each
// where eight CTAs do, so that two share an SM (8192 x 12288 bf16 backward: 162 us
// where two of 384 threads take 193), else of up to 512.
struct Variant {
  int vectors, threads, ctas;       // threads: 32, or a CTA's; ctas: 0: too wide
};
inline Variant variant_of(int64_t cols, bool bf16, int mode, int most, int threads) {
  const int e = bf16 ? 8 : 4, one = bf16 ? 1 : 2, lanes = mode == SHIFT ? PAYLOAD : 32;
  const int64_t slots = ceil_div(cols, e) + (mode == ALIGNED ? 0 : 1);   // unaligned rows end in 16 bytes more
  for (int n = one; n <= most * one; n += one)
    if (slots <= n * lanes) return {n, 32, 1};
  const int64_t warps = ceil_div(slots, (int64_t)2 * one * lanes);
  if (warps * 32 <= threads) return {2 * one, (int)warps * 32, 1};
  const int64_t ctas = warps <= 8 * MOST_CTAS ? ceil_div(warps, 8) : MOST_CTAS, each = ceil_div(warps, ctas) * 32;
  return each <= 512 ? Variant{2 * one, (int)each, (int)ctas} : Variant{2 * one, 0, 0};
}
// The gradient's: bf16 rows of four vectors a lane would leave an SM eight warps.
inline Variant grad_variant_of(int64_t cols, bool bf16, int mode) { return variant_of(cols, bf16, mode, bf16 ? 3 : 4, 512); }
// CTAs of the gradient kernel at most: each leaves a row of partial sums, so a CTA takes four rows (a row a warp: rounds of eight) at least where
// that leaves one for each SM.
inline int64_t grad_ctas(int64_t rows, bool warp_rows) {
  int64_t units = warp_rows ? ceil_div(rows, WARPS) : rows;
  if (units < 8) units = rows < 8 ? rows : 8;   // one for each place that a row may begin at
  const int64_t few = ceil_div(units, 4) > SMS ? ceil_div(units, 4) : SMS, most = 8 * SMS;
  const int64_t n = few < most ? few : most;
  return units < n ? units : n;
}
// Clusters of the gradient kernel at most: of three CTAs or more, two an SM.
inline int64_t grad_clusters(int64_t rows) { return rows < 2 * SMS / 3 ? rows : 2 * SMS / 3; }
inline int64_t wide_parts(int64_t rows) { return rows < 8 * 32 ? ceil_div(rows, 8) : 32; }
// Rows of partial sums of a variant at most.
inline int64_t parts_of(int64_t rows, const Variant& v) {
  return v.ctas == 0 ? wide_parts(rows) : v.ctas > 1 ? grad_clusters(rows) : grad_ctas(rows, v.threads == 32);
}

// Launches a persistent kernel with as many CTAs (clusters of `ctas`) as fit the SMs, `most` at most; their number, or -1.
template <auto KERNEL, class Arg>
int64_t launch(const Arg& a, int wvec, int threads, int ctas, int smem, int64_t most, bool by_eight, cudaStream_t s) {
  static std::atomic<int> resident[33][MOST_CTAS + 1];   // of this kernel on all SMs, by warps and ctas
  // for the current device, whichever that is
  if (smem > 47 * 1024 && cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -1;
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)ctas;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  c.gridDim = dim3((unsigned)ctas);
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = (size_t)smem;
  c.stream = s;
  c.attrs = &cluster;
  c.numAttrs = ctas > 1;
  std::atomic<int>& known = resident[threads / 32][ctas];
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t e = ctas > 1 ? cudaOccupancyMaxActiveClusters(&n, KERNEL, &c) : cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, smem);
    if (e != cudaSuccess || n < 1) return -1;
    if (ctas == 1) n *= (int)SMS;
    known.store(n, std::memory_order_relaxed);
  }
  int64_t grid = n < most ? n : most;
  if (by_eight && grid > 8) grid -= grid % 8;
  if (by_eight && grid < 8 && grid < most) return -1;   // a CTA (cluster) for each place that a row may begin at
  c.gridDim.x = (unsigned)(grid * ctas);
  return cudaLaunchKernelEx(&c, KERNEL, a, wvec) == cudaSuccess ? grid : -1;
}

// How the rows of matrices with these first addresses and pitches (elements) lie.
inline int mode_of(int64_t cols, int size, std::initializer_list<std::pair<const void*, int64_t>> all) {
  const int e = 16 / size;
  const auto first = *all.begin();
  bool aligned = cols % 8 == 0, same = true;
  for (const auto& m : all) {
    aligned = aligned && aligned16(m.first) && m.second % e == 0;
    same = same && (reinterpret_cast<uintptr_t>(m.first) - reinterpret_cast<uintptr_t>(first.first)) % 16 == 0 && (m.second - first.second) % e == 0;
  }
  return aligned ? ALIGNED : same ? PHASE : SHIFT;
}

template <bool BX, bool BW, int NV, int MAX_THREADS, bool CLUSTER = false>
int64_t forward_variant(const advopt_layer_norm_args& a, const Variant& v, int mode, int wvec, cudaStream_t s) {
  constexpr bool WARP = MAX_THREADS == 32;
  const int threads = WARP ? WARPS * 32 : v.threads;
  const int64_t most = WARP ? ceil_div(a.rows, WARPS) : a.rows;
  const int smem = Rows<BX, NV, ALIGNED, FWD_STAGES>::slots_of(threads) * 16;
  if (mode == ALIGNED) return launch<forward_kernel<BX, BW, NV, MAX_THREADS, ALIGNED, CLUSTER>>(a, wvec, threads, v.ctas, smem, most, false, s);
  if (mode == PHASE) return launch<forward_kernel<BX, BW, NV, MAX_THREADS, PHASE, CLUSTER>>(a, wvec, threads, v.ctas, smem, most, !WARP, s);
  return launch<forward_kernel<BX, BW, NV, MAX_THREADS, SHIFT, CLUSTER>>(a, wvec, threads, v.ctas, smem, most, false, s);
}

template <bool BX, bool BW>
int forward(const advopt_layer_norm_args& a, cudaStream_t s) {
  const int mode = mode_of(a.cols, BX ? 2 : 4, {{a.x, a.rows > 1 ? a.ldx : a.cols}, {a.y, a.cols}});
  const bool vec = mode == ALIGNED;
  const int wvec = aligned16(a.weight) && aligned16(a.bias);
  constexpr int N = BX ? 1 : 2;
  const Variant v = variant_of(a.cols, BX, mode, 4, 1024);
  int64_t n = 1;
  // many aligned bf16 rows: reading them thrice costs less than the clusters' barriers (1024 x 65536: 91 us for 109, 3276 x
  // 20480 94 for 94; float32 171 for 143, 188 for 129; 25 x 65536 bf16 12.6 for 6.8)
  const bool again = v.ctas == 0 || (BX && vec && v.ctas > 1 && a.rows > 2 * SMS);
  if (again) wide_forward_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
  else if (v.ctas > 1 && v.threads > 256) n = forward_variant<BX, BW, 2 * N, 512, true>(a, v, mode, wvec, s);
  else if (v.ctas > 1) n = forward_variant<BX, BW, 2 * N, 256, true>(a, v, mode, wvec, s);
  else if (v.threads > 512) n = forward_variant<BX, BW, 2 * N, 1024>(a, v, mode, wvec, s);
  else if (v.threads > 384) n = forward_variant<BX, BW, 2 * N, 512>(a, v, mode, wvec, s);
  else if (v.threads > 256) n = forward_variant<BX, BW, 2 * N, 384>(a, v, mode, wvec, s);
  else if (v.threads > 32) n = forward_variant<BX, BW, 2 * N, 256>(a, v, mode, wvec, s);
  else if (v.vectors == 4 * N) n = forward_variant<BX, BW, 4 * N, 32>(a, v, mode, wvec, s);
  else if (v.vectors == 3 * N) n = forward_variant<BX, BW, 3 * N, 32>(a, v, mode, wvec, s);
  else if (v.vectors == 2 * N) n = forward_variant<BX, BW, 2 * N, 32>(a, v, mode, wvec, s);
  else n = forward_variant<BX, BW, N, 32>(a, v, mode, wvec, s);
  const cudaError_t e = cudaGetLastError();
  return n < 0 ? set_error(ADVOPT_E_CUDA, "advopt_layer_norm: the kernel's attributes") : check_cuda(e, "advopt_layer_norm");
}

template <bool BX, bool BW, int NV, int MAX_THREADS, bool CLUSTER = false>
int64_t grad_variant(const advopt_layer_norm_grad_args& a, const Variant& v, int mode, int wvec, cudaStream_t s) {
  constexpr bool WARP = MAX_THREADS == 32;
  const int threads = WARP ? WARPS * 32 : v.threads;
  const int64_t ctas = WARP && mode != PHASE ? ceil_div(a.rows, WARPS) : a.rows, parts = parts_of(a.rows, v);
  const int64_t most = ctas < parts ? ctas : parts;
  const auto bytes = [&](int rows) { return 2 * rows * Rows<BX, NV, ALIGNED, grad_stages(BX)>::slots_of(threads) * 16; };
  if (mode == ALIGNED) return launch<grad_kernel<BX, BW, NV, MAX_THREADS, ALIGNED, CLUSTER>>(a, wvec, threads, v.ctas, bytes(grad_rows(BX, MAX_THREADS, ALIGNED)), most, false, s);
  if constexpr (MAX_THREADS != 320) {
    const int smem = bytes(grad_rows(BX, MAX_THREADS, SHIFT));
    if (mode == PHASE) return launch<grad_kernel<BX, BW, NV, MAX_THREADS, PHASE, CLUSTER>>(a, wvec, threads, v.ctas, smem, most, true, s);
    return launch<grad_kernel<BX, BW, NV, MAX_THREADS, SHIFT, CLUSTER>>(a, wvec, threads, v.ctas, smem, most, false, s);
  }
  return -1;
}

template <bool BX, bool BW>
int grad(const advopt_layer_norm_grad_args& a, cudaStream_t s) {
  const int64_t ldx = a.rows > 1 ? a.ldx : a.cols, lddy = a.rows > 1 ? a.lddy : a.cols;
  const int mode = a.dx ? mode_of(a.cols, BX ? 2 : 4, {{a.x, ldx}, {a.dy, lddy}, {a.dx, a.cols}}) : mode_of(a.cols, BX ? 2 : 4, {{a.x, ldx}, {a.dy, lddy}});
  const bool vec = mode == ALIGNED;
  const int wvec = aligned16(a.weight);
  constexpr int N = BX ? 1 : 2;
  const Variant v = grad_variant_of(a.cols, BX, mode);
  int64_t parts = 0;
  if (v.ctas == 0) {
    parts = wide_parts(a.rows);
    if (a.dx) wide_dx_kernel<BX, BW><<<(unsigned)(a.rows < 2 * SMS ? a.rows : 2 * SMS), 1024, 0, s>>>(a, vec, wvec);
    if (a.work) wide_sums_kernel<BX><<<dim3((unsigned)ceil_div(a.cols, 256), (unsigned)parts), 256, 0, s>>>(a, vec);
  } else if (v.ctas > 1) {
    parts = v.threads > 256 ? grad_variant<BX, BW, 2 * N, 512, true>(a, v, mode, wvec, s) : grad_variant<BX, BW, 2 * N, 256, true>(a, v, mode, wvec, s);
  } else if (v.threads > 384) {
    parts = grad_variant<BX, BW, 2 * N, 512>(a, v, mode, wvec, s);
  } else if (BX && mode == ALIGNED && v.threads > 256 && v.threads <= 320) {
    if constexpr (BX) parts = grad_variant<BX, BW, 2 * N, 320>(a, v, mode, wvec, s);
  } else if (v.threads > 256) {
    parts = grad_variant<BX, BW, 2 * N, 384>(a, v, mode, wvec, s);
  } else if (v.threads > 32) {
    parts = grad_variant<BX, BW, 2 * N, 256>(a, v, mode, wvec, s);
  } else if (v.vectors == 4 * N) {
    if constexpr (!BX) parts = grad_variant<BX, BW, 4 * N, 32>(a, v, mode, wvec, s);
  } else if (v.vectors == 3 * N) {
    parts = grad_variant<BX, BW, 3 * N, 32>(a, v, mode, wvec, s);
  } else if (v.vectors == 2 * N) {
    parts = grad_variant<BX, BW, 2 * N, 32>(a, v, mode, wvec, s);
  } else {
    parts = grad_variant<BX, BW, N, 32>(a, v, mode, wvec, s);
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
  int64_t parts = 0;   // whatever the rows' type and alignment
  for (const bool bf16 : {false, true})
    for (const int mode : {ln::ALIGNED, ln::PHASE, ln::SHIFT}) {
      const int64_t n = ln::parts_of(rows, ln::grad_variant_of(cols, bf16, mode));
      parts = parts < n ? n : parts;
    }
  return parts * 2 * cols * 4;
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
