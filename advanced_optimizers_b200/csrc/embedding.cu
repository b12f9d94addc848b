// Token embedding: y_t = scale * W[id_t], and its gradient
// dW_v = scale * sum of dy_t over the tokens t with id_t = v.
//
// Forward: a gather, bound by HBM (touched rows read once, y written once: 8192
// x 4096 bf16 17.7 us).
//
// Gradient: bound by HBM too (dy read once, every row of dW written once, of
// which most are zeros: 8192 x 4096 of 128256 bf16 172 us, 140 of them for 1.05
// GB of zeros).  The tokens are put in order of their ids first (a stable radix
// sort, so that the order of a row's sum follows from the ids alone); then each
// warp takes 8 or 32 tokens of that order, for 16 bytes a lane, and sums and
// writes, from registers, the rows that begin among them (25 us).  A row that
// fills a whole such chunk, and so may be of any length, leaves a float32
// partial sum in each of its chunks, and a further launch adds these up in
// order (7 us).  No float atomics: results repeat bit for bit.  Few tokens take
// one launch that compares instead of sorting.
#include <cooperative_groups.h>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "rows.cuh"

namespace advopt {
namespace emb {

namespace cg = cooperative_groups;

// An id as it is compared and sorted: `vocab` stands for all that contribute nothing.
__device__ __forceinline__ uint32_t key_of(const void* ids, bool wide, int64_t t, uint32_t vocab, int64_t padding) {
  const int64_t id = wide ? static_cast<const int64_t*>(ids)[t] : (int64_t) static_cast<const int32_t*>(ids)[t];
  return id < 0 || id >= (int64_t)vocab || id == padding ? vocab : (uint32_t)id;
}

// ---- forward: a warp per token and 1024 columns ----
constexpr int FWD_COLS = 1024;

template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) gather_kernel(const __grid_constant__ advopt_embedding_args a, uint32_t per_row) {
  const int lane = threadIdx.x & 31;
  const int64_t units = a.tokens * per_row;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (int64_t)gridDim.x * 8) {
    const int64_t t = per_row == 1 ? u : units >> 32 ? u / per_row : (int64_t)((uint32_t)u / per_row);
    const int64_t c0 = (u - t * per_row) * FWD_COLS;
    const uint32_t id = key_of(a.ids, a.id_bytes == 8, t, (uint32_t)a.vocab, -1);
    const bool good = id < (uint32_t)a.vocab;
    if (!good && lane == 0 && a.err) *reinterpret_cast<volatile int32_t*>(a.err) = 1;
    const int64_t from = good ? (int64_t)id * a.ldw : 0, to = t * a.width;
    const float nan = u2f(0x7fc00000u);
    if (VEC) {
      Oct<BF16> v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = c0 + (i * 32 + lane) * 8;
        if (c < a.width && good) v[i].load(a.weight, from + c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = c0 + (i * 32 + lane) * 8;
        if (c >= a.width) break;
        if (!good || a.scale != 1.0f) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = good ? __fmul_rn(v[i].at(e), a.scale) : nan;
          v[i].set(f);
        }
        v[i].store(a.y, to + c);
      }
    } else {
      const int64_t end = a.width < c0 + FWD_COLS ? a.width : c0 + FWD_COLS;
#pragma unroll 8
      for (int64_t c = c0 + lane; c < end; c += 32) {
        if (BF16) {
          const float f = good ? __fmul_rn(bf16_to_f(__ldg(static_cast<const uint16_t*>(a.weight) + from + c)), a.scale) : nan;
          static_cast<uint16_t*>(a.y)[to + c] = (uint16_t)f_to_bf16_rne(f);
        } else {
          static_cast<float*>(a.y)[to + c] = good ? __fmul_rn(__ldg(static_cast<const float*>(a.weight) + from + c), a.scale) : nan;
        }
      }
    }
  }
}

// ---- the gradient ----
struct Grad {
  void* dw;
  const void* dy;
  const void* ids;
  uint32_t* keys[2];        // ids and positions, from one buffer to the other at each pass
  uint32_t* at[2];
  float* part;              // [chunks][2][width]: of the row that a chunk begins in, and of the one that it ends in
  int64_t width;
  int64_t padding;
  uint32_t tokens, vocab;
  int wide, passes;
  float scale;
};

constexpr int CLUSTER = 8;             // CTAs that sort
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int BITS = 9, BINS = 1 << BITS;
constexpr int AHEAD = 8;               // tokens of a lane whose loads are on their way
constexpr int SORT_SMEM = (SORT_WARPS * BINS + 2 * BINS + SORT_WARPS) * 4;
constexpr int FILL_THREADS = 512, FILL = 4;   // 16-byte stores of a thread that writes zeros

// The lanes of `live` with this lane's digit, bit by bit (65536 tokens of a
// vocabulary of 50257: 36 us for the sort, with __match_any_sync 42).
__device__ __forceinline__ uint32_t peers_of(uint32_t d, uint32_t live) {
  uint32_t peers = live;
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const bool bit = (d >> b) & 1u;
    const uint32_t v = __ballot_sync(0xffffffffu, bit);
    peers &= bit ? v : ~v;
  }
  return peers;
}

// One cluster sorts, beside the kernel that writes the zeros: the sort reads and
// writes a few hundred KB that stay in L2, and takes less time than the zeros
// of a large table (16 us for 8192 tokens, two passes).
//
// A pass: every warp counts the digits of its contiguous share, the counts are
// summed over the digits, CTAs and warps before it, and the warp walks its share
// again, in order, and places each token behind those of its digit that came
// before.
__device__ __forceinline__ void sort_cluster(const Grad& g, uint32_t* sm) {
  cg::cluster_group cluster = cg::this_cluster();
  uint32_t* hist = sm;                                  // [SORT_WARPS][BINS]
  uint32_t* total = sm + SORT_WARPS * BINS;             // [BINS] of this CTA
  uint32_t* base = total + BINS;                        // [BINS] where this CTA's tokens of a digit begin
  uint32_t* warp_sums = base + BINS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster.block_rank();
  const uint32_t T = g.tokens;
  // a warp's share: whole 32s
  const uint32_t share = ((T + 32 * CLUSTER * SORT_WARPS - 1) / (32 * CLUSTER * SORT_WARPS)) * 32;
  const uint64_t first = (uint64_t)(rank * SORT_WARPS + warp) * share;
  const uint32_t begin = first < T ? (uint32_t)first : T;
  const uint32_t end = first + share < T ? (uint32_t)(first + share) : T;
  uint32_t* mine = hist + warp * BINS;
  for (int pass = 0; pass < g.passes; ++pass) {
    const uint32_t* from = g.keys[(pass + 1) & 1];
    const uint32_t* from_at = g.at[(pass + 1) & 1];
    uint32_t* to = g.keys[pass & 1];
    uint32_t* to_at = g.at[pass & 1];
    const int shift = pass * BITS;
    for (int i = lane; i < BINS; i += 32) mine[i] = 0;
    __syncwarp();
    for (uint32_t i0 = begin; i0 < end; i0 += 32 * AHEAD) {
      uint32_t key[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t i = i0 + k * 32 + lane;
        key[k] = 0;
        if (i < end) key[k] = pass ? from[i] : key_of(g.ids, g.wide, i, g.vocab, g.padding);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t i = i0 + k * 32 + lane;
        const uint32_t live = __ballot_sync(0xffffffffu, i < end);
        if (live == 0) break;
        const uint32_t d = (key[k] >> shift) & (BINS - 1), peers = peers_of(d, live);
        if (i < end && lane == __ffs(peers) - 1) mine[d] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    if (tid < BINS) {
      uint32_t sum = 0;
      for (int w = 0; w < SORT_WARPS; ++w) {
        const uint32_t n = hist[w * BINS + tid];
        hist[w * BINS + tid] = sum;
        sum += n;
      }
      total[tid] = sum;
    }
    cluster.sync();
    uint32_t all = 0, before = 0, upto = 0;
    if (tid < BINS) {
      for (uint32_t r = 0; r < CLUSTER; ++r) {
        const uint32_t n = cluster.map_shared_rank(total, r)[tid];
        before += r < rank ? n : 0u;
        all += n;
      }
      upto = all;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      if (lane == 31) warp_sums[warp] = upto;
    }
    __syncthreads();
    if (tid < BINS) {
      for (int w = 0; w < warp; ++w) upto += warp_sums[w];
      base[tid] = upto - all + before;
    }
    __syncthreads();
    for (uint32_t i0 = begin; i0 < end; i0 += 32 * AHEAD) {
      uint32_t key[AHEAD], from_place[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t i = i0 + k * 32 + lane;
        key[k] = from_place[k] = 0;
        if (i < end) {
          key[k] = pass ? from[i] : key_of(g.ids, g.wide, i, g.vocab, g.padding);
          from_place[k] = pass ? from_at[i] : i;
        }
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint32_t i = i0 + k * 32 + lane;
        const uint32_t live = __ballot_sync(0xffffffffu, i < end);
        if (live == 0) break;
        const uint32_t d = (key[k] >> shift) & (BINS - 1), peers = peers_of(d, live);
        if (i < end) {
          const uint32_t place = base[d] + mine[d] + __popc(peers & ((1u << lane) - 1u));
          to[place] = key[k];
          to_at[place] = from_place[k];
        }
        __syncwarp();
        if (i < end && lane == __ffs(peers) - 1) mine[d] += __popc(peers);
        __syncwarp();
      }
    }
    cluster.sync();   // the pass's tokens are in place for all CTAs, and `total` has been read
  }
}

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(SORT_THREADS) order_kernel(const __grid_constant__ Grad g) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the zeros do not wait for the order
  extern __shared__ uint32_t sm[];
  sort_cluster(g, sm);
}

// Zeros for all of dw (16-byte aligned), beside the sort on the other SMs.  In
// the order of the CTAs the stores reach HBM at 7.4 TB/s, a grid's width apart
// at 6.0.  The grid ends behind the sort, since its last CTA waits for it.
template <bool BF16>
__global__ void __launch_bounds__(FILL_THREADS) zero_kernel(void* dw, int64_t bytes) {
  uint4* p = static_cast<uint4*>(dw);
  const int64_t n = bytes >> 4;
  int64_t i = (int64_t)blockIdx.x * (FILL_THREADS * FILL) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < FILL; ++k, i += FILL_THREADS)
    if (i < n) p[i] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x != gridDim.x - 1) return;
  const int tail = (int)(bytes & 15) / (BF16 ? 2 : 4);
  if (threadIdx.x < tail) {
    if (BF16) reinterpret_cast<uint16_t*>(p + n)[threadIdx.x] = 0;
    else reinterpret_cast<float*>(p + n)[threadIdx.x] = 0.0f;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// 16 bytes of a row: the columns of a lane.
template <bool BF16>
struct Cols {
  static constexpr int E = BF16 ? 8 : 4;
  uint32_t w[4];
  __device__ __forceinline__ float at(int e) const { return BF16 ? u2f((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16) : u2f(w[e & 3]); }
  __device__ __forceinline__ void get(const void* base, int64_t k, int nv, bool vec) {
    if (vec && nv == E) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + k * (BF16 ? 2 : 4)));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else if (BF16) {
      const uint16_t* p = static_cast<const uint16_t*>(base) + k;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (2 * i < nv ? (uint32_t)__ldg(p + 2 * i) : 0u) | (2 * i + 1 < nv ? (uint32_t)__ldg(p + 2 * i + 1) << 16 : 0u);
    } else {
      const uint32_t* p = static_cast<const uint32_t*>(base) + k;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = i < nv ? __ldg(p + i) : 0u;
    }
  }
};

template <bool BF16>
__device__ __forceinline__ void write_row(const Grad& g, uint32_t row, int64_t c, int nv, bool vec, const float (&acc)[Cols<BF16>::E]) {
  constexpr int E = Cols<BF16>::E;
  const int64_t k = (int64_t)row * g.width + c;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = __fmul_rn(acc[e], g.scale);
  if constexpr (BF16) {
    uint16_t* p = static_cast<uint16_t*>(g.dw) + k;
    if (vec && nv == E) {
      *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < nv) p[e] = (uint16_t)f_to_bf16_rne(v[e]);
    }
  } else {
    float* p = static_cast<float*>(g.dw) + k;
    if (vec && nv == E) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < nv) p[e] = v[e];
    }
  }
}

// Whether a row that crosses from one chunk to the next is a long one, which
// fills one of them: `first` is the first key of the one, `end` the last of the
// other (g.vocab where that is not whole).
__device__ __forceinline__ bool is_long(uint32_t row, uint32_t first, uint32_t end) { return first == row || end == row; }

template <int E>
__device__ __forceinline__ void write_part(float* part, int nv, bool vec, const float (&acc)[E]) {
  if (vec && nv == E) {
#pragma unroll
    for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(part + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < nv) part[e] = acc[e];
  }
}

constexpr int SUM_WARPS = 4;

// A warp: the rows that begin among CHUNK tokens in order, for 16 bytes a lane.  A row that goes on into the next chunk, but fills neither, is
// followed there; of one that does, each chunk's warp sums its own tokens.
template <bool BF16, uint32_t CHUNK>
__global__ void __launch_bounds__(SUM_WARPS * 32, 7) sums_kernel(const __grid_constant__ Grad g, uint32_t slabs, int vec) {
  const int lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * SUM_WARPS + (threadIdx.x >> 5);
  const uint32_t chunk = (uint32_t)(u / slabs);
  if ((int64_t)chunk * CHUNK >= g.tokens) return;
  const uint32_t first = chunk * CHUNK;
  constexpr int E = Cols<BF16>::E;
  const int64_t c = ((u - (int64_t)chunk * slabs) * 32 + lane) * E;
  const int nv = c >= g.width ? 0 : g.width - c < E ? (int)(g.width - c) : E;
  const uint32_t* keys = g.keys[(g.passes + 1) & 1];
  const uint32_t* at = g.at[(g.passes + 1) & 1];
  const uint32_t mine = first + lane, next = mine + CHUNK;
  const bool here = lane < CHUNK && mine < g.tokens, behind = lane < CHUNK && next < g.tokens;
  const uint32_t key = here ? keys[mine] : g.vocab, pos = here ? at[mine] : 0u;
  const uint32_t more = behind ? keys[next] : g.vocab, more_pos = behind ? at[next] : 0u;
  const uint32_t n = __popc(__ballot_sync(0xffffffffu, key < g.vocab));   // those that contribute come first
  if (n == 0) return;
  const uint32_t head = __shfl_sync(0xffffffffu, key, 0), tail = __shfl_sync(0xffffffffu, key, CHUNK - 1);
  // the row that comes from the chunk before: long, or summed there
  const bool comes = first && keys[first - 1] == head;
  const bool long_ahead = comes && is_long(head, keys[first - CHUNK], tail);
  uint32_t begin = 0;
  if (comes && !long_ahead) begin = __popc(__ballot_sync(0xffffffffu, key == head));
  // the row that goes on into the next one
  const bool goes = n == CHUNK && __shfl_sync(0xffffffffu, more, 0) == tail;
  const bool long_behind = goes && is_long(tail, head, __shfl_sync(0xffffffffu, more, CHUNK - 1));
  uint32_t end = n;
  if (goes && !long_behind && begin < n) end += __popc(__ballot_sync(0xffffffffu, more == tail));
  if (begin >= n) return;
  float acc[E] = {};
  uint32_t cur = __shfl_sync(0xffffffffu, key, begin);
  bool partial = long_ahead;
  float* part = g.part + (int64_t)chunk * 2 * g.width + c;
  constexpr int U = 8;   // tokens whose values are on their way
  for (uint32_t i0 = begin; i0 < end; i0 += U) {
    Cols<BF16> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t j = i0 + i;
      const uint32_t p0 = __shfl_sync(0xffffffffu, pos, j & (CHUNK - 1)), p1 = __shfl_sync(0xffffffffu, more_pos, j & (CHUNK - 1));
      if (j < end) v[i].get(g.dy, (int64_t)(j < CHUNK ? p0 : p1) * g.width + c, nv, vec);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t j = i0 + i;
      const uint32_t k0 = __shfl_sync(0xffffffffu, key, j & (CHUNK - 1));
      if (j >= end) break;
      const uint32_t k = j < CHUNK ? k0 : tail;
      if (k != cur) {
        if (partial) write_part(part, nv, vec, acc);
        else if (nv) write_row<BF16>(g, cur, c, nv, vec, acc);
        partial = false;
        cur = k;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = __fadd_rn(acc[e], v[i].at(e));
    }
  }
  // a long row's sum of this chunk: the second place where the row begins here
  if (partial) write_part(part, nv, vec, acc);
  else if (long_behind) write_part(part + g.width, nv, vec, acc);
  else if (nv) write_row<BF16>(g, cur, c, nv, vec, acc);
}

// The long rows: a CTA takes those that begin in JOIN chunks, for 128 columns,
// a warp each; of rows of more than FAR parts every warp adds a share, and the
// shares are added in order.
constexpr int JOIN = 8;
constexpr uint32_t FAR = 64;

__device__ __forceinline__ void add_parts(float (&s)[4], const Grad& g, uint32_t chunk, uint32_t begin, uint32_t end, int64_t c, int nv, bool vec) {
  // part 0 is in its chunk's second place, the others in their first
  const auto at = [&](uint32_t p) { return g.part + ((int64_t)(chunk + p) * 2 + (p == 0)) * g.width + c; };
  if (vec && nv == 4) {
#pragma unroll 8
    for (uint32_t p = begin; p < end; ++p) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(at(p)));
      s[0] = __fadd_rn(s[0], q.x);
      s[1] = __fadd_rn(s[1], q.y);
      s[2] = __fadd_rn(s[2], q.z);
      s[3] = __fadd_rn(s[3], q.w);
    }
  } else {
#pragma unroll 4
    for (uint32_t p = begin; p < end; ++p) {
      const float* q = at(p);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) s[e] = __fadd_rn(s[e], __ldg(q + e));
    }
  }
}

template <bool BF16>
__device__ __forceinline__ void write_sum(const Grad& g, uint32_t row, int64_t c, float sum) {
  sum = __fmul_rn(sum, g.scale);
  const int64_t k = (int64_t)row * g.width + c;
  if (BF16) static_cast<uint16_t*>(g.dw)[k] = (uint16_t)f_to_bf16_rne(sum);
  else static_cast<float*>(g.dw)[k] = sum;
}

template <bool BF16, uint32_t CHUNK>
__global__ void __launch_bounds__(JOIN * 32) join_kernel(const __grid_constant__ Grad g, uint32_t slabs) {
  __shared__ float red[JOIN][128];
  __shared__ uint32_t far_row[JOIN], far_parts[JOIN];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t slab = blockIdx.x % slabs, chunk0 = blockIdx.x / slabs * JOIN, chunk = chunk0 + warp;
  const uint32_t* keys = g.keys[(g.passes + 1) & 1];
  const uint32_t T = g.tokens;
  const uint64_t last = ((uint64_t)chunk + 1) * CHUNK - 1;   // the last token of the warp's chunk
  uint32_t row = g.vocab, parts = 0;
  if (last + 1 < T) {
    row = keys[last];
    const uint32_t head = keys[last + 1 - CHUNK];
    const bool begins = row < g.vocab && keys[last + 1] == row && (last < CHUNK || keys[last - CHUNK] != row) &&
                        is_long(row, head, last + CHUNK < T ? keys[last + CHUNK] : g.vocab);
    if (begins) {
      // the first token behind the row's, between lo and hi: each lane looks at one of 32 places between
      uint32_t lo = (uint32_t)last + 2, hi = T;
      while (lo < hi) {
        const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, at < hi && keys[at] == row));
        if (n == 0) break;
        const uint32_t reach = lo + n * step;
        lo += (n - 1) * step + 1;
        if (reach < hi) hi = reach;
      }
      parts = (lo - 1) / CHUNK - chunk + 1;   // this chunk's and the following ones'
    }
  }
  const bool far = parts > FAR;
  if (lane == 0) {
    far_row[warp] = row;
    far_parts[warp] = far ? parts : 0u;
  }
  const int64_t c = (int64_t)slab * 128 + lane * 4;
  const int nv = c >= g.width ? 0 : g.width - c < 4 ? (int)(g.width - c) : 4;
  const bool vec = (g.width & 3) == 0;   // the partial sums are 16-byte aligned
  if (parts && !far) {
    float s[4] = {};
    add_parts(s, g, chunk, 0, parts, c, nv, vec);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nv) write_sum<BF16>(g, row, c + e, s[e]);
  }
  if (!__syncthreads_or(far)) return;
  for (int b = 0; b < JOIN; ++b) {
    const uint32_t all = far_parts[b];
    if (all == 0) continue;
    const uint32_t each = (all + JOIN - 1) / JOIN, p0 = warp * each < all ? warp * each : all, p1 = p0 + each < all ? p0 + each : all;
    float s[4] = {};
    add_parts(s, g, chunk0 + b, p0, p1, c, nv, vec);
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][lane * 4 + e] = s[e];
    __syncthreads();
    const int64_t mine = (int64_t)slab * 128 + threadIdx.x;
    if (threadIdx.x < 128 && mine < g.width) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < JOIN; ++w) sum = __fadd_rn(sum, red[w][threadIdx.x]);
      write_sum<BF16>(g, far_row[b], mine, sum);
    }
    __syncthreads();
  }
}

// ---- few tokens: one launch, no order ----
// A CTA takes a run of rows of dw, finds among the ids which of them occur,
// and writes the others' zeros.  A warp then takes a row that occurs and 16
// bytes a lane, and adds the row's tokens as they come.
constexpr int FEW = 256;
constexpr int FEW_BYTES = 32768;       // of dw a CTA at most, about

template <bool BF16>
__global__ void __launch_bounds__(FEW) few_kernel(const __grid_constant__ Grad g, uint32_t rows, uint32_t wide, int vec) {
  constexpr int E = Cols<BF16>::E;
  __shared__ uint32_t ids[FEW];
  __shared__ uint32_t met[FEW_BYTES / 2 / 32];   // a bit for each of the CTA's rows
  __shared__ uint32_t list[FEW], found;          // the rows that occur
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t first = blockIdx.x * rows, here = g.vocab - first < rows ? g.vocab - first : rows;
  for (uint32_t i = threadIdx.x; i < (here + 31) / 32; i += FEW) met[i] = 0;
  const uint32_t key = threadIdx.x < g.tokens ? key_of(g.ids, g.wide, threadIdx.x, g.vocab, g.padding) : g.vocab;
  ids[threadIdx.x] = key;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  const uint32_t mine = key - first;
  if (key < g.vocab && mine < here && !(atomicOr(&met[mine >> 5], 1u << (mine & 31)) >> (mine & 31) & 1u))
    list[atomicAdd(&found, 1u)] = mine;   // in any order: each row's sum is its own
  __syncthreads();
  // `wide` vectors a row
  const float zero[E] = {};
  for (uint32_t u = threadIdx.x; u < here * wide; u += FEW) {
    const uint32_t row = u / wide;
    const int64_t c = (int64_t)(u - row * wide) * E;
    if (!(met[row >> 5] >> (row & 31) & 1u)) write_row<BF16>(g, first + row, c, g.width - c < E ? (int)(g.width - c) : E, vec, zero);
  }
  const uint32_t chunks = (wide + 31) / 32;
  for (uint32_t u = warp; u < found * chunks; u += FEW / 32) {
    const uint32_t row = first + list[u / chunks];
    const int64_t c = ((int64_t)(u % chunks) * 32 + lane) * E;
    const int nv = c >= g.width ? 0 : g.width - c < E ? (int)(g.width - c) : E;
    float acc[E] = {};
    for (uint32_t t0 = 0; t0 < g.tokens; t0 += 32) {
      uint32_t with = __ballot_sync(0xffffffffu, ids[t0 + lane] == row);   // beyond the last token: vocab
      while (with) {
        Cols<BF16> v[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (with) {
            v[i].get(g.dy, (int64_t)(t0 + __ffs(with) - 1) * g.width + c, nv, vec);
            with &= with - 1;
            n = i + 1;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = __fadd_rn(acc[e], v[i].at(e));
          }
      }
    }
    if (nv) write_row<BF16>(g, row, c, nv, vec, acc);
  }
}
inline bool is_few(int64_t tokens) { return tokens <= FEW; }

struct Work {
  int64_t list, part, bytes;   // bytes of one of the four lists, where the partial sums begin, all
};
// Chunks of 32 tokens, a lane's worth each, unless their warps are too few to
// hide each other's loads (16 an SM): a quarter of the tokens then takes a
// warp a quarter of the time (2048 x 2048 bf16: 7.5 + 5.9 us for the sums and
// the join, with 32 tokens 15.1 + 3.9; 8192 x 4096: 25 + 17, with 32 25 + 7).
inline int64_t chunk_of(int64_t tokens, int64_t width, int size) {
  return ceil_div(tokens, 32) * ceil_div(width * size, 512) <= 148 * 16 ? 8 : 32;
}
inline Work work_of(int64_t tokens, int64_t width, int64_t chunk) {
  const int64_t list = (tokens * 4 + 15) / 16 * 16;
  return {list, 4 * list, 4 * list + ceil_div(tokens, chunk) * 2 * width * 4};
}

template <bool BF16, uint32_t CHUNK>
void sums(const advopt_embedding_grad_args& a, const Grad& g, cudaStream_t s) {
  const int64_t chunks = ceil_div(a.tokens, CHUNK), slabs = ceil_div(a.width, 32 * Cols<BF16>::E);
  const int vec = aligned16(a.dy) && aligned16(a.dweight) && a.width % Cols<BF16>::E == 0;
  sums_kernel<BF16, CHUNK><<<(unsigned)ceil_div(chunks * slabs, SUM_WARPS), SUM_WARPS * 32, 0, s>>>(g, (uint32_t)slabs, vec);
  if (chunks > 1) {
    const int64_t wide = ceil_div(a.width, 128);
    join_kernel<BF16, CHUNK><<<(unsigned)(ceil_div(chunks, JOIN) * wide), JOIN * 32, 0, s>>>(g, (uint32_t)wide);
  }
}

template <bool BF16>
int grad(const advopt_embedding_grad_args& a, cudaStream_t s) {
  Grad g;
  const int64_t chunk = chunk_of(a.tokens, a.width, BF16 ? 2 : 4);
  const Work w = work_of(a.tokens, a.width, chunk);
  unsigned char* at = static_cast<unsigned char*>(a.work);
  g.dw = a.dweight;
  g.dy = a.dy;
  g.ids = a.ids;
  for (int i = 0; i < 2; ++i) {
    g.keys[i] = reinterpret_cast<uint32_t*>(at + 2 * i * w.list);
    g.at[i] = reinterpret_cast<uint32_t*>(at + (2 * i + 1) * w.list);
  }
  g.part = reinterpret_cast<float*>(at + w.part);
  g.width = a.width;
  g.padding = a.padding;
  g.tokens = (uint32_t)a.tokens;
  g.vocab = (uint32_t)a.vocab;
  g.wide = a.id_bytes == 8;
  g.scale = a.scale;
  g.passes = 1;
  while (a.vocab >> (g.passes * BITS)) ++g.passes;   // the keys are 0 .. vocab
  if (is_few(a.tokens)) {
    const int64_t row = a.width * (BF16 ? 2 : 4), wide = ceil_div(a.width, Cols<BF16>::E);
    // two CTAs an SM, of 512 bytes to 32 KB each
    int64_t share = a.vocab * row / (2 * 148);
    share = share < 512 ? 512 : share < FEW_BYTES ? share : FEW_BYTES;
    const int64_t rows = row >= share ? 1 : share / row;
    const int vec = aligned16(a.dy) && a.width % Cols<BF16>::E == 0;
    few_kernel<BF16><<<(unsigned)ceil_div(a.vocab, rows), FEW, 0, s>>>(g, (uint32_t)rows, (uint32_t)wide, vec);
    return check_cuda(cudaGetLastError(), "advopt_embedding_grad");
  }
  const int64_t bytes = a.vocab * a.width * (BF16 ? 2 : 4), zeros = ceil_div(bytes, FILL_THREADS * FILL * 16);
  const char* where = "advopt_embedding_grad";
  cudaError_t e = cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_SMEM);
  if (e != cudaSuccess) return check_cuda(e, where);
  order_kernel<<<CLUSTER, SORT_THREADS, SORT_SMEM, s>>>(g);
  e = cudaGetLastError();
  if (e != cudaSuccess) return check_cuda(e, where);
  cudaLaunchAttribute beside;
  beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)zeros);
  config.blockDim = dim3(FILL_THREADS);
  config.stream = s;
  config.attrs = &beside;
  config.numAttrs = 1;
  e = cudaLaunchKernelEx(&config, zero_kernel<BF16>, a.dweight, bytes);
  if (e != cudaSuccess) return check_cuda(e, where);
  if (chunk == 8) sums<BF16, 8>(a, g, s);
  else sums<BF16, 32>(a, g, s);
  return check_cuda(cudaGetLastError(), where);
}

template <bool BF16>
void forward(const advopt_embedding_args& a, cudaStream_t s) {
  const int64_t per_row = ceil_div(a.width, FWD_COLS), ctas = ceil_div(a.tokens * per_row, 8);
  const unsigned grid = (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
  const bool vec = aligned16(a.y) && aligned16(a.weight) && a.width % 8 == 0 && a.ldw * (BF16 ? 2 : 4) % 16 == 0;
  if (vec) gather_kernel<BF16, true><<<grid, 256, 0, s>>>(a, (uint32_t)per_row);
  else gather_kernel<BF16, false><<<grid, 256, 0, s>>>(a, (uint32_t)per_row);
}

constexpr int64_t LIMIT = (int64_t)1 << 31;

}  // namespace emb
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_embedding(const advopt_embedding_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->vocab < 0 || a->width < 0 || a->tokens >= emb::LIMIT || a->vocab >= emb::LIMIT ||
      a->width >= emb::LIMIT || (a->vocab > 1 && a->ldw < a->width) || (a->id_bytes != 4 && a->id_bytes != 8))
    return set_error(ADVOPT_E_INVALID, "advopt_embedding: bad arguments");
  if (!known_dtype(a->dtype)) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_embedding: float32 and bfloat16 are supported");
  if (a->tokens == 0 || a->width == 0) return ADVOPT_OK;
  if (!a->y || !a->ids || (a->vocab && !a->weight)) return set_error(ADVOPT_E_INVALID, "advopt_embedding: null pointer");
  if (a->dtype == ADVOPT_DT_BF16) emb::forward<true>(*a, static_cast<cudaStream_t>(stream));
  else emb::forward<false>(*a, static_cast<cudaStream_t>(stream));
  return check_cuda(cudaGetLastError(), "advopt_embedding");
}

extern "C" int64_t advopt_embedding_grad_work(int64_t tokens, int64_t width, int32_t dtype) {
  return emb::is_few(tokens) || width <= 0 ? 0 : emb::work_of(tokens, width, emb::chunk_of(tokens, width, bytes_of(dtype))).bytes;
}

extern "C" int advopt_embedding_grad(const advopt_embedding_grad_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->vocab < 0 || a->width < 0 || a->tokens >= emb::LIMIT || a->vocab >= emb::LIMIT ||
      a->width >= emb::LIMIT || (a->id_bytes != 4 && a->id_bytes != 8))
    return set_error(ADVOPT_E_INVALID, "advopt_embedding_grad: bad arguments");
  if (!known_dtype(a->dtype))
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_embedding_grad: float32 and bfloat16 are supported");
  if (a->vocab == 0 || a->width == 0) return ADVOPT_OK;
  if (!a->dweight || !aligned16(a->dweight) || (a->tokens && (!a->dy || !a->ids)) ||
      (!emb::is_few(a->tokens) && (!a->work || !aligned16(a->work))))
    return set_error(ADVOPT_E_INVALID, "advopt_embedding_grad: null or unaligned pointer");
  const int64_t chunks = ceil_div(a->tokens, 8);
  if (a->vocab > ((int64_t)1 << 43) / a->width || chunks * ceil_div(a->width, 128) / emb::SUM_WARPS >= emb::LIMIT - 1)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_embedding_grad: too many tokens or rows for this width");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == ADVOPT_DT_BF16 ? emb::grad<true>(*a, s) : emb::grad<false>(*a, s);
}
