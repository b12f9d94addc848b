// Token embedding: y_t = scale * W[id_t], and its gradient
// dW_v = scale * sum of dy_t over the tokens t with id_t = v.
//
// Forward: a gather, bound by HBM (touched rows read once, y written once).
//
// Gradient: bound by HBM too (dy read once, every row of dW written once, of
// which most are zeros).  The tokens are put in order of their ids first (a
// stable radix sort, so that the order of a row's sum follows from the ids
// alone); then each warp sums 32 tokens of that order for 256 columns in
// registers and writes the rows that begin and end among them.  A row that
// reaches over several such chunks leaves a float32 partial sum in each, and
// a third launch adds these up in order.  No atomics: results repeat bit for
// bit.
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
constexpr int SORT_SMEM = (SORT_WARPS * BINS + 2 * BINS + SORT_WARPS) * 4;
constexpr uint32_t CHUNK = 32;         // tokens of one warp, so that a lane holds one token's id

// One cluster sorts while the other ones write the zeros: the sort reads and
// writes a few hundred KB that stay in L2, and takes less time than the
// zeros of a large table.
//
// A pass of the sort: every warp counts the digits of its contiguous share,
// the counts are summed over the digits, CTAs and warps before it, and the
// warp walks its share again, in order, and places each token behind those of
// its digit that came before.
template <int UNUSED>
__device__ void sort_cluster(const Grad& g, uint32_t* sm) {
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
    for (uint32_t i = begin + lane; i - lane < end; i += 32) {
      const uint32_t live = __ballot_sync(0xffffffffu, i < end);
      if (i < end) {
        const uint32_t key = pass ? from[i] : key_of(g.ids, g.wide, i, g.vocab, g.padding);
        const uint32_t d = (key >> shift) & (BINS - 1);
        const uint32_t peers = __match_any_sync(live, d);
        if (lane == __ffs(peers) - 1) mine[d] += __popc(peers);
      }
      __syncwarp();
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
    for (uint32_t i = begin + lane; i - lane < end; i += 32) {
      const uint32_t live = __ballot_sync(0xffffffffu, i < end);
      if (i < end) {
        const uint32_t key = pass ? from[i] : key_of(g.ids, g.wide, i, g.vocab, g.padding);
        const uint32_t d = (key >> shift) & (BINS - 1);
        const uint32_t peers = __match_any_sync(live, d);
        const uint32_t place = base[d] + mine[d] + __popc(peers & ((1u << lane) - 1u));
        to[place] = key;
        to_at[place] = pass ? from_at[i] : i;
        __syncwarp(live);
        if (lane == __ffs(peers) - 1) mine[d] += __popc(peers);
      }
      __syncwarp();
    }
    cluster.sync();   // the pass's tokens are in place for all CTAs, and `total` has been read
  }
}

template <bool BF16>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(SORT_THREADS) order_kernel(const __grid_constant__ Grad g) {
  extern __shared__ uint32_t sm[];
  if (blockIdx.x < CLUSTER) {
    sort_cluster<0>(g, sm);
    return;
  }
  // zeros: dw is 16-byte aligned
  const int64_t bytes = (int64_t)g.vocab * g.width * (BF16 ? 2 : 4);
  uint4* p = static_cast<uint4*>(g.dw);
  const int64_t n = bytes >> 4, stride = (int64_t)(gridDim.x - CLUSTER) * SORT_THREADS;
  const int64_t i0 = (int64_t)(blockIdx.x - CLUSTER) * SORT_THREADS + threadIdx.x;
  for (int64_t i = i0; i < n; i += stride) p[i] = make_uint4(0, 0, 0, 0);
  const int tail = (int)(bytes & 15) / (BF16 ? 2 : 4);
  if (i0 < tail) {
    if (BF16) reinterpret_cast<uint16_t*>(p + n)[i0] = 0;
    else reinterpret_cast<float*>(p + n)[i0] = 0.0f;
  }
}

template <bool BF16>
__device__ __forceinline__ void write_row(const Grad& g, uint32_t row, int64_t c, int nv, bool vec, const float (&acc)[8]) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(acc[e], g.scale);
  Oct<BF16> o;
  o.set(v);
  o.put(g.dw, (int64_t)row * g.width + c, nv, vec);
}

// A warp: CHUNK tokens in order x 256 columns, eight a lane.
template <bool BF16>
__global__ void __launch_bounds__(256) sums_kernel(const __grid_constant__ Grad g, uint32_t slabs, int vec) {
  const int lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t chunk = (uint32_t)(u / slabs);
  const uint32_t first = chunk * CHUNK;
  if ((int64_t)chunk * CHUNK >= g.tokens) return;
  const int64_t c = (int64_t)(u - (int64_t)chunk * slabs) * 256 + lane * 8;
  const int nv = c >= g.width ? 0 : g.width - c < 8 ? (int)(g.width - c) : 8;
  const uint32_t* keys = g.keys[(g.passes + 1) & 1];
  const uint32_t* at = g.at[(g.passes + 1) & 1];
  const uint32_t key = first + lane < g.tokens ? keys[first + lane] : g.vocab;
  const uint32_t pos = first + lane < g.tokens ? at[first + lane] : 0u;
  const uint32_t n = __popc(__ballot_sync(0xffffffffu, key < g.vocab));   // those that contribute come first
  if (n == 0) return;
  const uint32_t ahead = first ? keys[first - 1] : g.vocab;
  const uint32_t behind = first + CHUNK < g.tokens ? keys[first + CHUNK] : g.vocab;
  float acc[8] = {};
  uint32_t cur = __shfl_sync(0xffffffffu, key, 0);
  bool open_ahead = cur == ahead;
  float* part = g.part + (int64_t)chunk * 2 * g.width + c;
  constexpr int U = 8;
  for (uint32_t i0 = 0; i0 < n; i0 += U) {
    Oct<BF16> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t p = __shfl_sync(0xffffffffu, pos, i0 + i);
      if (i0 + i < n) v[i].get(g.dy, (int64_t)p * g.width + c, nv, vec);
      else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t k = __shfl_sync(0xffffffffu, key, i0 + i);
      if (i0 + i >= n) break;
      if (k != cur) {
        if (open_ahead) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < nv) part[e] = acc[e];
          open_ahead = false;
        } else if (nv) {
          write_row<BF16>(g, cur, c, nv, vec, acc);
        }
        cur = k;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = __fadd_rn(acc[e], v[i].at(e));
    }
  }
  if (open_ahead || (n == CHUNK && cur == behind)) {
    if (!open_ahead) part += g.width;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < nv) part[e] = acc[e];
  } else if (nv) {
    write_row<BF16>(g, cur, c, nv, vec, acc);
  }
}

// The rows that reach over chunks: a CTA looks at 32 chunks for those that
// begin in them, for 128 columns.  The partial sums of a row are split over
// the warps in order, and the warps' sums are added in order.
constexpr int JOIN_WARPS = 16;

template <bool BF16>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const __grid_constant__ Grad g, uint32_t slabs) {
  __shared__ float red[JOIN_WARPS][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t slab = blockIdx.x % slabs, group = blockIdx.x / slabs;
  const uint32_t* keys = g.keys[(g.passes + 1) & 1];
  const uint32_t T = g.tokens;
  const uint64_t last = ((uint64_t)group * 32 + lane + 1) * CHUNK - 1;   // the last token of this lane's chunk
  uint32_t key = g.vocab;
  bool begins = false;
  if (last + 1 < T) {
    key = keys[last];
    begins = key < g.vocab && keys[last + 1] == key && (last < CHUNK || keys[last - CHUNK] != key);
  }
  uint32_t todo = __ballot_sync(0xffffffffu, begins);
  const int64_t c = (int64_t)slab * 128 + lane * 4;
  const int nv = c >= g.width ? 0 : g.width - c < 4 ? (int)(g.width - c) : 4;
  while (todo) {
    const int b = __ffs(todo) - 1;
    todo &= todo - 1;
    const uint32_t row = __shfl_sync(0xffffffffu, key, b);
    const uint32_t chunk = group * 32 + b;
    // the first token behind the row's
    uint32_t lo = (chunk + 1) * CHUNK, hi = T;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (keys[mid] > row) hi = mid;
      else lo = mid + 1;
    }
    const uint32_t parts = (lo - 1) / CHUNK - chunk + 1;   // this chunk's and the following ones'
    const uint32_t each = (parts + JOIN_WARPS - 1) / JOIN_WARPS;
    const uint32_t p0 = warp * each < parts ? warp * each : parts, p1 = p0 + each < parts ? p0 + each : parts;
    float s[4] = {};
    for (uint32_t p = p0; p < p1; ++p) {
      // part 0 is what the chunk ends in, the others what they begin in
      const float* from = g.part + ((int64_t)(chunk + p) * 2 + (p == 0)) * g.width + c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) s[e] = __fadd_rn(s[e], from[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][lane * 4 + e] = s[e];
    __syncthreads();
    if (threadIdx.x < 128 && (int64_t)slab * 128 + threadIdx.x < g.width) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < JOIN_WARPS; ++w) sum = __fadd_rn(sum, red[w][threadIdx.x]);
      sum = __fmul_rn(sum, g.scale);
      const int64_t k = (int64_t)row * g.width + (int64_t)slab * 128 + threadIdx.x;
      if (BF16) static_cast<uint16_t*>(g.dw)[k] = (uint16_t)f_to_bf16_rne(sum);
      else static_cast<float*>(g.dw)[k] = sum;
    }
    __syncthreads();
  }
}

struct Work {
  int64_t list, part, bytes;   // bytes of one of the four lists, where the partial sums begin, all
};
inline Work work_of(int64_t tokens, int64_t width) {
  const int64_t list = (tokens * 4 + 15) / 16 * 16;
  return {list, 4 * list, 4 * list + ceil_div(tokens, CHUNK) * 2 * width * 4};
}

template <bool BF16>
int grad(const advopt_embedding_grad_args& a, cudaStream_t s) {
  Grad g;
  const Work w = work_of(a.tokens, a.width);
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
  const int64_t trip = SORT_THREADS * 16 * 4, zeros = ceil_div(a.vocab * a.width * (BF16 ? 2 : 4), trip);
  const int64_t most = 2 * 148 - CLUSTER;
  const int64_t fill = ceil_div(zeros < most ? zeros : most, CLUSTER) * CLUSTER;
  cudaError_t e = cudaFuncSetAttribute(order_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_SMEM);
  if (e != cudaSuccess) return check_cuda(e, "advopt_embedding_grad");
  order_kernel<BF16><<<(unsigned)(CLUSTER + fill), SORT_THREADS, SORT_SMEM, s>>>(g);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.tokens == 0) return check_cuda(e, "advopt_embedding_grad");
  const int64_t chunks = ceil_div(a.tokens, CHUNK), slabs = ceil_div(a.width, 256);
  const int vec = aligned16(a.dy) && aligned16(a.dweight) && a.width * (BF16 ? 2 : 4) % 16 == 0 && a.width % 8 == 0;
  sums_kernel<BF16><<<(unsigned)ceil_div(chunks * slabs, 8), 256, 0, s>>>(g, (uint32_t)slabs, vec);
  if (chunks > 1) {
    const int64_t wide = ceil_div(a.width, 128);
    join_kernel<BF16><<<(unsigned)(ceil_div(chunks, 32) * wide), JOIN_WARPS * 32, 0, s>>>(g, (uint32_t)wide);
  }
  return check_cuda(cudaGetLastError(), "advopt_embedding_grad");
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

extern "C" int64_t advopt_embedding_grad_work(int64_t tokens, int64_t width) {
  return tokens <= 0 || width <= 0 ? 0 : emb::work_of(tokens, width).bytes;
}

extern "C" int advopt_embedding_grad(const advopt_embedding_grad_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->vocab < 0 || a->width < 0 || a->tokens >= emb::LIMIT || a->vocab >= emb::LIMIT ||
      a->width >= emb::LIMIT || (a->id_bytes != 4 && a->id_bytes != 8))
    return set_error(ADVOPT_E_INVALID, "advopt_embedding_grad: bad arguments");
  if (!known_dtype(a->dtype))
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_embedding_grad: float32 and bfloat16 are supported");
  if (a->vocab == 0 || a->width == 0) return ADVOPT_OK;
  if (!a->dweight || !aligned16(a->dweight) || (a->tokens && (!a->dy || !a->ids || !a->work || !aligned16(a->work))))
    return set_error(ADVOPT_E_INVALID, "advopt_embedding_grad: null or unaligned pointer");
  const int64_t chunks = ceil_div(a->tokens, emb::CHUNK);
  if (chunks * ceil_div(a->width, 256) / 8 >= emb::LIMIT - 1 || ceil_div(chunks, 32) * ceil_div(a->width, 128) >= emb::LIMIT)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_embedding_grad: too many tokens for this width");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->dtype == ADVOPT_DT_BF16 ? emb::grad<true>(*a, s) : emb::grad<false>(*a, s);
}
