// Block-scaled 8-bit product for sm_100a:
//   D = residual + dropout(sum_b 2^(sa + sb) sum_{k in block b} A B^T + bias)
//
// Operands are K-major e4m3 / e5m2 with one power-of-two scale (E8M0) for
// each 128 elements along K; the tensor cores apply the scales themselves
// (tcgen05.mma kind::mxf8f6f4 with block scales), so the accumulator never
// leaves tensor memory until the product is done.  The hardware's scale
// granule is 32 elements: one 32-bit scale word per row holds the scales of
// four consecutive 128-blocks, and the four K = 32 instructions of a block all
// name that block's byte, so no scale is replicated in memory.
//
// One CTA computes a 128 x BN tile: "rows" come from one operand (the
// accumulator's 128 lanes), "columns" from the other.  With few tokens the
// operands trade places (`swap`): the weights fill the 128 lanes and BN
// shrinks to the tokens.  With few tiles, S CTAs of a cluster split K and add
// their accumulators through distributed shared memory, in rank order.
//   * warp 0: TMA loads of 128-byte wide K blocks, 128B swizzle;
//   * warp 1: copies scale words to tensor memory (tcgen05.cp) and issues the
//     MMAs;
//   * warps 2 and 3: gather the scale words of four blocks at a time;
//   * then all eight warps: the epilogue.
// With many tiles, pairs of CTAs walk them persistently (further down).
// Every wait is bounded and gives up when another role has; the CTA then
// waits (bounded) for its copies and MMAs in flight, frees its tensor memory
// and reports through *err.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>

#include "advopt.h"
#include "capi_internal.h"
#include "common.cuh"
#include "drop.cuh"
#include "fp8_ring.cuh"

namespace advopt {
namespace fp8 {

constexpr int BM = 128, BK = 128;
constexpr int THREADS = 256;
constexpr int SMS = 148, PAIRS = SMS / 2;
constexpr int SF_SLOTS = 4;                   // scale words of 4 x 4 blocks in flight
constexpr int SF_SLOT_BYTES = 512 * 3;        // rows, columns 0..127, columns 128..255
// float32 results of long K are summed in chunks of at most CHUNK blocks, each a
// product of its own, which are added in float32 and in order: the tensor cores
// truncate as they accumulate, an error that grows with K.  A chunk of 64 blocks
// is low by 5e-7 of the result in the Frobenius norm (normal values; 7e-7 with
// columns ten times as large; a product that rounds: 1.5e-7), and so is a sum of
// chunks; uncut, 128 blocks are off by 1.2e-6 and 980 by 1.8e-5.  bf16 results
// round at 2^-9 and do without.
// The pairs' epilogue adds its chunks to D.  Single CTAs split K over a cluster
// and keep a CTA's chunks in accumulators of their own, long_accs of them; a
// longer sum takes a launch for each as many, which adds to D.
constexpr int CHUNK = 64;
constexpr int long_accs(int bn) { return bn <= 64 ? 7 : bn <= 128 ? 3 : 1; }

// One operand as the kernel sees it.
struct Side {
  const uint8_t* scales;
  int64_t ld;
  int64_t extent;     // rows
  int shift;          // 7: a scale row per 128 rows, 0: per row
  int code;
};

struct GemmArgs {
  Side p, q;          // accumulator lanes / columns
  void* d;
  const void* bias;
  const void* residual;
  int64_t ldd, ldres, n;
  int kblocks;
  int swap;           // D[q][p] instead of D[p][q]
  int vec;            // rows of D and the residual are 16-byte aligned
  int vec_bias;
  int drop;
  int more;           // LONG: D holds the sum of the blocks before these
  int32_t* err;
};

// LONG: float32 sums of more than CHUNK blocks a CTA, in as many accumulators as
// tensor memory has room for.
template <int BN, bool LONG>
struct Cfg {
  static constexpr int STAGES = BN >= 256 || BN <= 32 ? 4 : 6;
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SF_OFF = STAGES * STAGE_BYTES;
  static constexpr int SMEM = SF_OFF + SF_SLOTS * SF_SLOT_BYTES + 1024;
  static constexpr int SF_BUFS = 2;   // scale buffers in tensor memory
  static constexpr int SF_COLS = 4 + (BN > 128 ? 8 : 4);
  static constexpr int ACCS = LONG ? long_accs(BN) : 1;
  static constexpr int SF_COL = ACCS * BN;
  static constexpr int USED = SF_COL + SF_BUFS * SF_COLS;
  static constexpr uint32_t TMEM = USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(USED <= (BN <= 32 ? 256 : 512), "two CTAs share an SM's tensor memory at BN = 32");
};

// Instruction descriptor of kind::mxf8f6f4 with E8M0 scales, K-major operands.
__device__ __forceinline__ uint32_t instr_desc(int rows, int cols, int a_code, int b_code) {
  return ((uint32_t)a_code << 7) | ((uint32_t)b_code << 10) | ((uint32_t)(cols >> 3) << 17) | (1u << 23) |
         ((uint32_t)(rows >> 4) << 24);
}
// ... and which byte of the scale words it takes, for both operands.
__device__ __forceinline__ constexpr uint32_t sf_id(uint32_t j) { return (j << 4) | (j << 29); }

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// The four K = 32 steps of one staged block and the commit that frees the stage
// (of both CTAs of a pair).  One asm statement with the predicate inside: all
// lanes reach it together, so descriptors stay in uniform registers.  As four
// calls under a branch on the elected lane, 8192 x 14336 x 4096 took 424 us
// instead of 375.
#define ADVOPT_FP8_BLOCK(GROUP, COMMIT)                                                                              \
  "{\n .reg .pred p, q, t;\n .reg .b32 al, bl;\n .reg .b64 a, b;\n"                                              \
  " setp.ne.b32 q, %9, 0;\n setp.ne.b32 p, %6, 0;\n setp.eq.b32 t, 0, 0;\n"                                       \
  " mov.b64 a, {%1, %8};\n mov.b64 b, {%2, %8};\n"                                                                 \
  " @q tcgen05.mma.cta_group::" GROUP ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], p;\n"   \
  " add.u32 al, %1, 2;\n add.u32 bl, %2, 2;\n mov.b64 a, {al, %8};\n mov.b64 b, {bl, %8};\n"                     \
  " @q tcgen05.mma.cta_group::" GROUP ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], t;\n"   \
  " add.u32 al, %1, 4;\n add.u32 bl, %2, 4;\n mov.b64 a, {al, %8};\n mov.b64 b, {bl, %8};\n"                     \
  " @q tcgen05.mma.cta_group::" GROUP ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], t;\n"   \
  " add.u32 al, %1, 6;\n add.u32 bl, %2, 6;\n mov.b64 a, {al, %8};\n mov.b64 b, {bl, %8};\n"                     \
  " @q tcgen05.mma.cta_group::" GROUP ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], t;\n"   \
  " @q tcgen05.commit.cta_group::" GROUP COMMIT "\n}\n"
template <bool PAIR>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate, uint64_t* freed, uint32_t hi, uint32_t one) {
  if (PAIR)
    asm volatile(
        ADVOPT_FP8_BLOCK("2", ".mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%7], %10;")
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(smem_u32(freed)), "r"(hi),
        "r"(one), "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        ADVOPT_FP8_BLOCK("1", ".mbarrier::arrive::one.shared::cluster.b64 [%7];")
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(smem_u32(freed)), "r"(hi),
        "r"(one)
        : "memory");
}
#undef ADVOPT_FP8_BLOCK

// 32 rows of 16 bytes -> 4 tensor-memory columns, repeated for the four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc, uint32_t one) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n}\n"
               ::"r"(taddr), "l"(desc), "r"(one)
               : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t one) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n"
      ::"r"(smem_u32(bar)), "r"(one)
      : "memory");
}

// 32 accumulator columns of a lane's row.  The values are there after
// tmem_wait32, which names them so that no use moves before it.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");
}

// r += 32 columns of another accumulator, in float32.
__device__ __forceinline__ void add_columns(uint32_t taddr, uint32_t (&r)[32]) {
  uint32_t t[32];
  tmem_ld32(taddr, t);
  tmem_wait32(t);
#pragma unroll
  for (int e = 0; e < 32; ++e) r[e] = f2u(__fadd_rn(u2f(r[e]), u2f(t[e])));
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait of a whole warp that also gives up once another role has; all
// lanes get the same answer, so that they stay together afterwards.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < (1u << 22); ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 255u) == 255u && __any_sync(0xffffffffu, *abort_flag)) return false;
  }
  return false;
}

// One lane of a converged warp.  The issuing warps run their loops with all
// lanes, so that addresses, descriptors and counters stay in uniform registers,
// and only the copies and MMAs themselves are predicated: with the loops inside
// `if (lane == 0)`, 8192 x 14336 x 4096 took 480 us instead of 424.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// A position in a ring of N barriers: slot, and the parity of its use.
template <int N>
struct Ring {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// A matrix descriptor's high half; the low half is the address and counts up in 16-byte units.
__device__ __forceinline__ uint64_t desc_at(uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; }
constexpr uint32_t TILE_HI = (1024u >> 4) | (1u << 14) | (2u << 29);    // 1024 bytes between 8-row groups, 128-byte swizzle
constexpr uint32_t SCALE_HI = (128u >> 4) | (1u << 14);                  // 128 bytes between 8-row groups, none
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4); }

// The product is launched while the kernel before it in the stream may still
// run (programmatic dependent launch): barriers and tensor memory are set up
// meanwhile, and nothing is read or written before that kernel's results are
// there.  The kernel after it may start its own set-up as early.
__device__ __forceinline__ void after_earlier_kernels() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_float(uint32_t saddr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
  return v;
}

__device__ __forceinline__ float4 peer_float4(uint32_t saddr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote));
  return v;
}

// Scale word (four consecutive K blocks) of row r; rows outside get 1.
__device__ __forceinline__ uint32_t scale_word(const Side& s, int64_t r, int group) {
  if (r >= s.extent) return 0x7F7F7F7Fu;
  return __ldg(reinterpret_cast<const uint32_t*>(s.scales + (r >> s.shift) * s.ld) + group);
}

// One group's scale words of a tile, four rows a lane.
template <int BN>
struct ScaleWords {
  static constexpr int PARTS = 1 + (BN + 127) / 128;
  uint32_t w[PARTS][4];
  __device__ __forceinline__ void load(const GemmArgs& g, int64_t p0, int64_t q0, int group, int lane) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[0][e] = scale_word(g.p, p0 + 32 * e + lane, group);
#pragma unroll
    for (int c = 1; c < PARTS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[c][e] = scale_word(g.q, q0 + 128 * (c - 1) + 32 * e + lane, group);
  }
  // row 32 e + l goes to 16-byte line l, word e: what the copy to tensor memory takes
  __device__ __forceinline__ void store(unsigned char* slot, int lane) const {
#pragma unroll
    for (int c = 0; c < PARTS; ++c)
      *reinterpret_cast<uint4*>(slot + 512 * c + 16 * lane) = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
};

// Swapped operands: W tokens (columns) of feature p, one of D's columns per lane.
template <bool BF16, bool LONG, int W>
__device__ __forceinline__ void emit(const GemmArgs& g, const DropSpec& d, uint32_t step, int64_t p, int64_t q0,
                                     float (&v)[W]) {
  if (p >= g.p.extent || q0 >= g.q.extent) return;
  const int w = g.q.extent - q0 < W ? (int)(g.q.extent - q0) : W;
  const float b = !g.bias ? 0.0f
                  : BF16  ? bf16_to_f(static_cast<const uint16_t*>(g.bias)[p])
                          : static_cast<const float*>(g.bias)[p];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (j >= w) break;
    float x = v[j];
    if (LONG && g.more) x = __fadd_rn(static_cast<const float*>(g.d)[(q0 + j) * g.ldd + p], x);
    if (g.bias) x = __fadd_rn(x, b);
    if (g.drop) x = drop1(x, d, step, (uint64_t)((q0 + j) * g.n + p));
    if (g.residual)
      x = __fadd_rn(x, BF16 ? bf16_to_f(static_cast<const uint16_t*>(g.residual)[(q0 + j) * g.ldres + p])
                            : static_cast<const float*>(g.residual)[(q0 + j) * g.ldres + p]);
    if (BF16) static_cast<uint16_t*>(g.d)[(q0 + j) * g.ldd + p] = (uint16_t)bf16x2(x, 0.0f);
    else static_cast<float*>(g.d)[(q0 + j) * g.ldd + p] = x;
  }
}

// A warp's 32 x 32 block, a row per lane, turned through shared memory (4 KB of
// the warp's own) so that four lanes hold a row's 32 columns: D, the residual
// and the bias are then touched in whole sectors, and one Philox evaluation
// serves a lane's eight elements.  With a row per lane the epilogue took as
// long as the MMAs of K = 4096 (16.5k cycles a tile).
// 16-byte piece c of row r lies at c ^ (r & 7): stores and loads touch all banks.
__device__ __forceinline__ void turn_in(unsigned char* turn, const uint32_t (&r)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(turn + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
  __syncwarp();
}

// A block at D's edge, or of a D whose rows are not 16-byte aligned: a column
// per lane and a row at a time, so that what a warp touches is still contiguous
// (with eight columns a lane, 333 x 2041 took 29 us instead of 10).
__device__ __forceinline__ float turned(const unsigned char* turn, int r, int lane) {
  return *reinterpret_cast<const float*>(turn + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2));
}
template <bool BF16>
__device__ __noinline__ void store_edge(void* d, int64_t ldd, const unsigned char* turn, int rows, int cols) {
  const int lane = threadIdx.x & 31;
  if (lane < cols) {
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 8) {
      float x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = turned(turn, r0 + r, lane);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < rows) {
          if (BF16) static_cast<uint16_t*>(d)[(r0 + r) * ldd + lane] = (uint16_t)bf16x2(x[r], 0.0f);
          else static_cast<float*>(d)[(r0 + r) * ldd + lane] = x[r];
        }
    }
  }
  __syncwarp();
}
// A lane's 32 keep bits of a block: row 8 i + lane / 4, columns 8 (lane % 4) ..
__device__ __forceinline__ uint32_t block_mask(const GemmArgs& g, const DropSpec& d, uint32_t step, int64_t p0, int64_t q0) {
  const int lane = threadIdx.x & 31;
  const int64_t p = p0 + (lane >> 2), q = q0 + 8 * (lane & 3);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= drop_bits8(d, step, (uint64_t)((p + 8 * i) * g.n + q)) << (8 * i);
  return bits;
}
// mask: block_mask's, a lane's own word, where g.drop.
template <bool BF16>
__device__ __noinline__ void emit_edge(const GemmArgs& g, const DropSpec& d, uint32_t mask, const unsigned char* turn,
                                       int64_t p0, int64_t q0, bool more, bool last) {
  const int lane = threadIdx.x & 31;
  const int64_t q = q0 + lane;
  const int rows = g.p.extent - p0 < 32 ? (int)(g.p.extent - p0) : 32;
  const bool in = q < g.q.extent;
  const bool drop = g.drop && last, add = g.residual && last && in, biased = g.bias && last && in;
  const float bias = !biased ? 0.0f
                     : BF16  ? bf16_to_f(static_cast<const uint16_t*>(g.bias)[q])
                             : static_cast<const float*>(g.bias)[q];
  const int64_t ldd = g.ldd, ldres = g.ldres;
  char* at = static_cast<char*>(g.d) + (p0 * ldd + q) * (BF16 ? 2 : 4);
  const char* res = static_cast<const char*>(g.residual) + (p0 * ldres + q) * (BF16 ? 2 : 4);
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 8) {
    float x[8], t[8], s[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const bool live = in && r0 + r < rows;
      t[r] = !(add && live) ? 0.0f
             : BF16         ? bf16_to_f(reinterpret_cast<const uint16_t*>(res)[(r0 + r) * ldres])
                            : reinterpret_cast<const float*>(res)[(r0 + r) * ldres];
      s[r] = !BF16 && more && live ? reinterpret_cast<const float*>(at)[(r0 + r) * ldd] : 0.0f;
      x[r] = turned(turn, r0 + r, lane);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (!BF16 && more) x[r] = __fadd_rn(s[r], x[r]);
      if (biased) x[r] = __fadd_rn(x[r], bias);
      if (drop) {
        // this element's bit is with the lane that holds its row and eight columns in block_mask's order
        const uint32_t word = __shfl_sync(0xffffffffu, mask, r * 4 + (lane >> 3));
        x[r] = (word >> (r0 + (lane & 7))) & 1u ? __fmul_rn(x[r], d.scale) : 0.0f;
      }
      if (add) x[r] = __fadd_rn(x[r], t[r]);
      if (in && r0 + r < rows) {
        if (BF16) reinterpret_cast<uint16_t*>(at)[(r0 + r) * ldd] = (uint16_t)bf16x2(x[r], 0.0f);
        else reinterpret_cast<float*>(at)[(r0 + r) * ldd] = x[r];
      }
    }
  }
  __syncwarp();
}

// EXTRA: there may be a bias, a dropout or a residual.  Without one the code
// between a block's loads and its stores is short.  mask: the block's keep bits
// (block_mask), where they were drawn before.
template <bool BF16, bool EXTRA>
__device__ __forceinline__ void emit_block(const GemmArgs& g, const DropSpec& d, uint32_t step, const unsigned char* turn,
                                           int64_t p0, int64_t q0, bool more, bool last, const uint32_t* mask = nullptr) {
  if (p0 >= g.p.extent || q0 >= g.q.extent) {
    __syncwarp();
    return;
  }
  if (!g.vec || q0 + 32 > g.q.extent) {
    if (more || (EXTRA && last && (g.bias || g.drop || g.residual))) {
      const uint32_t bits = !(EXTRA && g.drop && last) ? 0u : mask ? mask[threadIdx.x & 31] : block_mask(g, d, step, p0, q0);
      emit_edge<BF16>(g, d, bits, turn, p0, q0, more, last);
    } else {
      const int64_t at = p0 * g.ldd + q0, rows = g.p.extent - p0, cols = g.q.extent - q0;
      store_edge<BF16>(BF16 ? (void*)(static_cast<uint16_t*>(g.d) + at) : (void*)(static_cast<float*>(g.d) + at), g.ldd, turn,
                       rows < 32 ? (int)rows : 32, cols < 32 ? (int)cols : 32);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const int part = lane & 3;
  const int64_t p = p0 + (lane >> 2), q = q0 + 8 * part;
  // the four rows' loads go out together and first: the way through shared
  // memory and the masks take as long as they do.  The last rows may lie behind
  // the matrix.
  bool in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) in[i] = p + 8 * i < g.p.extent;
  constexpr int LINES = BF16 ? 1 : 2;
  uint4 res[4][LINES];
  float bias[8];
  if (EXTRA && last) {
    if (g.residual) {
      const char* at = static_cast<const char*>(g.residual) + (p * g.ldres + q) * (BF16 ? 2 : 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < LINES; ++h)
          res[i][h] = in[i] ? __ldg(reinterpret_cast<const uint4*>(at + 8 * i * g.ldres * (BF16 ? 2 : 4)) + h) : uint4{};
    }
    if (g.bias) load8<BF16>(g.bias, q, 8, g.vec_bias, bias);
  }
  uint32_t keep = 0;
  if (EXTRA && last && g.drop) keep = mask ? mask[lane] : block_mask(g, d, step, p0, q0);
  float v[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    const float4 a = *reinterpret_cast<const float4*>(turn + row * 128 + (((2 * part) ^ (row & 7)) << 4));
    const float4 b = *reinterpret_cast<const float4*>(turn + row * 128 + (((2 * part + 1) ^ (row & 7)) << 4));
    v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
    v[i][4] = b.x; v[i][5] = b.y; v[i][6] = b.z; v[i][7] = b.w;
  }
  __syncwarp();
  if (!BF16 && more) {
    const float* at = static_cast<const float*>(g.d) + p * g.ldd + q;
    float4 f[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i][0] = in[i] ? *reinterpret_cast<const float4*>(at + 8 * i * g.ldd) : float4{};
      f[i][1] = in[i] ? *reinterpret_cast<const float4*>(at + 8 * i * g.ldd + 4) : float4{};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float t[8] = {f[i][0].x, f[i][0].y, f[i][0].z, f[i][0].w, f[i][1].x, f[i][1].y, f[i][1].z, f[i][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(t[e], v[i][e]);
    }
  }
  if (EXTRA && last) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (g.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(v[i][e], bias[e]);
      }
      if (g.drop) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = (keep >> (8 * i + e)) & 1u ? __fmul_rn(v[i][e], d.scale) : 0.0f;
      }
      if (g.residual) {
        const uint4& a = res[i][0];
        const uint4& b = res[i][LINES - 1];
        if (BF16) {
          const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(v[i][e], u2f((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16));
        } else {
          const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(v[i][e], u2f(w[e]));
        }
      }
    }
  }
  if (BF16) {
    uint16_t* out = static_cast<uint16_t*>(g.d) + p * g.ldd + q;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in[i]) *reinterpret_cast<uint4*>(out + 8 * i * g.ldd) = make_uint4(bf16x2(v[i][0], v[i][1]), bf16x2(v[i][2], v[i][3]),
                                                                  bf16x2(v[i][4], v[i][5]), bf16x2(v[i][6], v[i][7]));
  } else {
    float* out = static_cast<float*>(g.d) + p * g.ldd + q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!in[i]) continue;
      *reinterpret_cast<float4*>(out + 8 * i * g.ldd) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
      *reinterpret_cast<float4*>(out + 8 * i * g.ldd + 4) = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
    }
  }
}

// Brings a tile of the residual towards L2, a row per lane.
__device__ __forceinline__ void prefetch_rows(const void* base, int64_t ld, int es, int64_t row, int64_t rows, int64_t col,
                                              int64_t cols, int width) {
  if (row >= rows) return;
  const char* p = static_cast<const char*>(base) + (row * ld + col) * es;
  const int bytes = (int)(cols - col < width ? cols - col : width) * es;
  for (int b = 0; b < bytes; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
}

// One 128 x BN tile, split over the S CTAs of a cluster along K.
// LONG is a kernel of its own: its branches and its tensor memory cost the
// others 0.1 to 0.2 us.
template <int BN, int S, bool BF16, bool LONG>
__global__ void __launch_bounds__(THREADS, BN <= 32 ? 2 : 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                const __grid_constant__ GemmArgs g, const __grid_constant__ DropSpec d) {
  using C = Cfg<BN, LONG>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES / 2], empty[C::STAGES], sf_full[SF_SLOTS], sf_empty[SF_SLOTS], acc_full;
  __shared__ uint32_t tmem_base, masks[4][BN / 32][32];
  __shared__ int abort_flag, loads_issued;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const uint32_t rank = S > 1 ? cluster_rank() : 0u;
  const int64_t tile = blockIdx.x / S;
  const int64_t p_tiles = (g.p.extent + BM - 1) / BM;
  const int64_t p0 = (tile % p_tiles) * BM, q0 = (tile / p_tiles) * BN;
  // this CTA's K blocks: whole groups of four, so that scale words are not split
  const int groups = (g.kblocks + 3) / 4;
  const int kb0 = 4 * (int)((int64_t)groups * rank / S);
  const int kb1 = min(g.kblocks, 4 * (int)((int64_t)groups * (rank + 1) / S));
  const int nkb = kb1 > kb0 ? kb1 - kb0 : 0;
  // LONG: accumulators, and blocks in each (whole groups of four)
  const int accs = LONG ? (nkb + CHUNK - 1) / CHUNK : 1;
  const int chunk = LONG && nkb ? ((nkb + accs - 1) / accs + 3) / 4 * 4 : 4;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      if (s % 2 == 0) mbar_init(&full[s / 2], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SF_SLOTS; ++s) {
      mbar_init(&sf_full[s], 32);
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    abort_flag = 0;
    loads_issued = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(C::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  after_earlier_kernels();
  // through a warp reduction: it lands in a uniform register, where the MMAs want it
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, tmem_base);

  if (warp == 0) {
    const bool one = elect_one();
    Ring<C::STAGES> st;
    int issued = 0;
    for (int i = 0; i < nkb; ++i, st.next()) {
      if (i >= C::STAGES && !wait_warp(&empty[st.slot], st.phase ^ 1u, abort_v)) {
        abort_flag = 1;
        break;
      }
      if (one) {
        unsigned char* sp = smem + st.slot * C::STAGE_BYTES;
        uint64_t* bar = &full[st.slot >> 1];
        if ((i & 1) == 0) mbar_arrive_tx(bar, i + 1 < nkb ? 2 * C::STAGE_BYTES : C::STAGE_BYTES);
        tma_load_2d(sp, &map_p, (kb0 + i) * BK, (int)p0, bar);
        tma_load_2d(sp + C::A_BYTES, &map_q, (kb0 + i) * BK, (int)q0, bar);
      }
      __syncwarp();
      issued = i + 1;
    }
    if (one) loads_issued = issued;
    // the commits' last arrivals have come before this CTA's shared memory goes
    // to another: each slot's latest use
    for (int i = nkb > C::STAGES ? nkb - C::STAGES : 0; i < nkb && issued == nkb; ++i)
      if (!wait_warp(&empty[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, abort_v)) {
        abort_flag = 1;
        break;
      }
  } else if (warp == 1) {
    const bool one = elect_one();
    const uint32_t tiles_lo = desc_lo(smem_u32(smem)), sf_lo = desc_lo(smem_u32(smem + C::SF_OFF));
    const uint32_t idesc = instr_desc(BM, BN, g.p.code, g.q.code);
    Ring<C::STAGES / 2> st;
    Ring<SF_SLOTS> sf;
    uint32_t acc = tmem;
    int next = 0;   // LONG: the block that the next accumulator starts with
    bool ok = true;
    for (int i = 0, grp = 0; i < nkb && ok; i += 4, ++grp) {
      const uint32_t sfp = tmem + C::SF_COL + (uint32_t)(grp % C::SF_BUFS) * C::SF_COLS, sfq = sfp + 4;
      if (LONG && i == next) {
        next += chunk;
        acc += i ? BN : 0;
      }
      ok = wait_warp(&sf_full[sf.slot], sf.phase, abort_v);
      // this buffer's last readers, the MMAs of SF_BUFS groups ago, are done
      if (ok && grp >= C::SF_BUFS) ok = wait_warp(&sf_empty[(grp - C::SF_BUFS) % SF_SLOTS],
                                                      (uint32_t)((grp - C::SF_BUFS) / SF_SLOTS) & 1u, abort_v);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t src = sf_lo + sf.slot * (SF_SLOT_BYTES / 16);
      copy_scales(sfp, desc_at(src, SCALE_HI), one);
      copy_scales(sfq, desc_at(src + 32, SCALE_HI), one);
      if (BN > 128) copy_scales(sfq + 4, desc_at(src + 64, SCALE_HI), one);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        if (i + j < nkb && ok) {
          ok = wait_warp(&full[st.slot], st.phase, abort_v);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (i + j + h < nkb) {
              const uint32_t lo = tiles_lo + (2 * st.slot + h) * (C::STAGE_BYTES / 16);
              mma_block<false>(acc, lo, lo + C::A_BYTES / 16, idesc | sf_id(j + h), sfp, sfq,
                               LONG ? i + j + h + chunk > next : i + j + h > 0,
                               &empty[2 * st.slot + h], TILE_HI, one);
            }
          }
          st.next();
        }
      }
      // the last groups' buffers are not written again: an arrival that no one waits for could come after this
      // CTA's shared memory went to another (waiting for them cost 1 x 4096 x 4096 0.25 us of 6.9)
      mma_commit(&sf_empty[sf.slot], one && i + 4 * C::SF_BUFS < nkb);
      sf.next();
    }
    if (!ok) abort_flag = 1;
    // also when giving up: the commit tells when everything issued is done
    mma_commit(&acc_full, one);
  } else if (warp < 4) {
    // warps 2 and 3 take the groups in turn, each loading its next one before it stores the present one
    bool ok = true;
    ScaleWords<BN> now, then;
    int grp = warp - 2;
    if (4 * grp < nkb) now.load(g, p0, q0, (kb0 >> 2) + grp, lane);
    for (; 4 * grp < nkb; grp += 2) {
      const int slot = grp % SF_SLOTS;
      if (4 * (grp + 2) < nkb) then.load(g, p0, q0, (kb0 >> 2) + grp + 2, lane);
      if (grp >= SF_SLOTS) ok = wait_warp(&sf_empty[slot], (uint32_t)(grp / SF_SLOTS - 1) & 1u, abort_v);
      if (!ok) {
        abort_flag = 1;
        break;
      }
      now.store(smem + C::SF_OFF + slot * SF_SLOT_BYTES, lane);
      mbar_arrive(&sf_full[slot]);
      now = then;
    }
  } else {
    // warps 4..7 have no part in the main loop: meanwhile they bring the
    // residual near and draw the masks of the blocks this CTA will write
    // (1000 x 2048 x 2048 bf16 with a dropout: 8.2 us, drawn in the epilogue 15.4)
    const int quarter = warp & 3;
    if (g.residual) {
      if (!g.swap) prefetch_rows(g.residual, g.ldres, BF16 ? 2 : 4, p0 + quarter * 32 + lane, g.p.extent, q0, g.q.extent, BN);
      else
        for (int j = threadIdx.x - 128; j < BN; j += 128)
          prefetch_rows(g.residual, g.ldres, BF16 ? 2 : 4, q0 + j, g.q.extent, p0, g.p.extent, BM);
    }
    if (g.drop && !g.swap) {
      const uint32_t step = drop_step(d);
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c)
        if (S == 1 || (4 * c + quarter) % S == (int)rank)
          masks[quarter][c][lane] = block_mask(g, d, step, p0 + quarter * 32, q0 + 32 * c);
    }
  }
  // the ring's warps are done: all eight share the epilogue
  __syncwarp();
  if (g.drop) __syncthreads();   // the masks
  const bool have = wait_warp(&acc_full, 0, abort_v);
  if (!have) abort_flag = 1;
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

  const uint32_t step = g.drop ? drop_step(d) : 0u;
  const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
  const bool extra = g.bias || g.drop || g.residual;
  const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16);
  if (S == 1) {
    if (have) {
#pragma unroll 1
      for (int c = 32 * half; c < BN; c += 64) {
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        tmem_wait32(r);
        if (LONG)
#pragma unroll 1
          for (int i = chunk; i < nkb; i += chunk) add_columns(taddr + i / chunk * BN + c, r);
        if (!g.swap) {
          // over the ring, which is drained once the accumulator is complete
          unsigned char* turn = smem + warp * 4096;
          turn_in(turn, r);
          if (extra) emit_block<BF16, true>(g, d, step, turn, p0 + quarter * 32, q0 + c, LONG && g.more, true, masks[quarter][c / 32]);
          else emit_block<BF16, false>(g, d, step, turn, p0 + quarter * 32, q0 + c, LONG && g.more, true);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[16 * h + e]);
            emit<BF16, LONG, 16>(g, d, step, p0 + row, q0 + c + 16 * h, v);
          }
        }
      }
    }
  } else {
    // over the ring, which is drained once the accumulator is complete.  Rank r
    // adds up columns r BN / S ..: swapped, [column][row] floats, a row (one of
    // D's columns) per lane; else the turned 32 x 32 blocks, so that D's rows
    // are written in whole sectors.
    float* acc = reinterpret_cast<float*>(smem);
    if (have) {
#pragma unroll 1
      for (int c = 32 * half; c < BN; c += 64) {
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        tmem_wait32(r);
        if (LONG)
#pragma unroll 1
          for (int i = chunk; i < nkb; i += chunk) add_columns(taddr + i / chunk * BN + c, r);
        if (!nkb)
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        if (g.swap) {
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[(c + e) * BM + row] = __uint_as_float(r[e]);
        } else {
          turn_in(smem + (c / 32 * 4 + quarter) * 4096, r);
        }
      }
    }
    __syncwarp();
    cluster_sync();
    if (have) {
      if (g.swap) {
        constexpr int PER = BN / S, W = PER < 16 ? PER / 2 : 8;
#pragma unroll 1
        for (int c = W * half; c < PER; c += 2 * W) {
          float v[W];
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const uint32_t at = smem_u32(acc + (rank * PER + c + e) * BM + row);
            v[e] = peer_float(at, 0);
#pragma unroll
            for (int o = 1; o < S; ++o) v[e] = __fadd_rn(v[e], peer_float(at, o));
          }
          emit<BF16, LONG, W>(g, d, step, p0 + row, q0 + rank * PER + c, v);
        }
      } else {
        // the tile's 4 BN / 32 blocks, dealt out to the cluster's 8 S warps
        constexpr int BLOCKS = 4 * BN / 32;
#pragma unroll 1
        for (int b = warp * S + (int)rank; b < BLOCKS; b += 8 * S) {
          unsigned char* turn = smem + b * 4096;
          unsigned char* own = smem + (BLOCKS + warp) * 4096;   // this block's sum
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            const uint32_t at = smem_u32(turn + (i * 32 + lane) * 16);
            float4 x = peer_float4(at, 0);
#pragma unroll
            for (int o = 1; o < S; ++o) {
              const float4 y = peer_float4(at, o);
              x = make_float4(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y), __fadd_rn(x.z, y.z), __fadd_rn(x.w, y.w));
            }
            *reinterpret_cast<float4*>(own + (i * 32 + lane) * 16) = x;
          }
          __syncwarp();
          if (extra) emit_block<BF16, true>(g, d, step, own, p0 + (b & 3) * 32, q0 + b / 4 * 32, LONG && g.more, true, masks[b & 3][b / 4]);
          else emit_block<BF16, false>(g, d, step, own, p0 + (b & 3) * 32, q0 + b / 4 * 32, LONG && g.more, true);
        }
      }
    }
    __syncwarp();
    cluster_sync();   // no CTA leaves while its shared memory is read
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (abort_flag) {
    // wait (bounded) for the loads and MMAs in flight before memory is given back
    if (threadIdx.x == 0) {
      for (int i = loads_issued > C::STAGES ? loads_issued - C::STAGES : 0; i < loads_issued; ++i)
        mbar_wait(&full[i % C::STAGES / 2], (uint32_t)(i / C::STAGES) & 1u, 1u << 20);
      mbar_wait(&acc_full, 0, 1u << 20);
      if (g.err) *reinterpret_cast<volatile int32_t*>(g.err) = 1;
    }
    __syncthreads();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
  }
}

// ---- many tiles: pairs of CTAs (cta_group::2), persistent, two accumulators ----
// A pair computes 256 x BN tiles: each CTA stages its 128 rows of P and half
// of Q's BN rows, so a staged byte feeds twice the multiplications of the
// single-CTA kernel; the even CTA issues the MMAs for both.  Each CTA's tensor
// memory holds its 128 rows of two accumulators.  At BN = 256 these and the
// scales do not fit 512 columns: the accumulators then share 32 columns, which
// the epilogue reads first, and the next tile's MMAs start once it has.
template <int BN>
struct PairCfg {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN / 2 * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 6;   // even: blocks are staged, and waited for, in twos
  static constexpr int SF_OFF = STAGES * STAGE_BYTES;
  static constexpr int TURN_OFF = SF_OFF + SF_SLOTS * SF_SLOT_BYTES;
  static constexpr int EPI = BN > 224 ? 4 : 8;   // epilogue warps: as many as there is shared memory to turn blocks in
  static constexpr int SMEM = TURN_OFF + EPI * 4096 + 1024;
  static constexpr int THREADS = 128 + 32 * EPI;
  static constexpr int SF_COLS = 4 + (BN > 128 ? 8 : 4);
  static constexpr int SF_BUFS = BN > 224 ? 2 : 3;
  static constexpr int SHARED = 2 * BN + SF_BUFS * SF_COLS > 512 ? 32 : 0;
  static constexpr int ACC_STRIDE = BN - SHARED;
  static constexpr int SF_COL = BN + ACC_STRIDE;
};

struct PairArgs {
  int p_tiles, q_tiles;   // of 256 and BN
  int band;
  int chunks, chunk_blocks;
};

__device__ __forceinline__ uint32_t map_to(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A load into this CTA that reports to the even CTA's barrier (no multicast).
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc, uint32_t one) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n @q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n}\n"
               ::"r"(taddr), "l"(desc), "r"(one)
               : "memory");
}
// Arrives at this barrier of both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint32_t one) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n"
      ::"r"(smem_u32(bar)), "h"((uint16_t)3), "r"(one)
      : "memory");
}
// Tile t: bands of `band` row tiles, walked row-fastest, so that the tiles in
// flight share both operands in L2.  Every band reads all of the column operand
// again, so bands are as tall as the operands of 74 tiles in flight stay within
// 40 MB of L2: 8192 x 14336 x 4096 takes 400 / 390 / 384 us in bands of 8 / 16 /
// 32 (under the power cap), 8192 x 4096 x 14336, where 8 hold 62 MB already,
// 392 / 412 / 435.
__device__ __forceinline__ void pair_origin(int t, const PairArgs& w, int bn, int64_t& p0, int64_t& q0) {
  const int band = t / (w.band * w.q_tiles), r = t - band * w.band * w.q_tiles;
  const int rows = min(w.band, w.p_tiles - band * w.band);
  p0 = (int64_t)(band * w.band + r % rows) * (2 * BM);
  q0 = (int64_t)(r / rows) * bn;
}

template <int BN, bool BF16, bool EXTRA>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg<BN>::THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                const __grid_constant__ GemmArgs g, const __grid_constant__ PairArgs w, const __grid_constant__ DropSpec d) {
  using C = PairCfg<BN>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES / 2], empty[C::STAGES], sf_full[SF_SLOTS], sf_empty[SF_SLOTS], acc_full[2], acc_empty[2];
  __shared__ uint64_t drain;
  __shared__ uint32_t tmem_base;
  __shared__ __align__(8) uint32_t loads[2][2];   // loads: the even CTA's, what each CTA's Fills ended with
  __shared__ int abort_flag;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int n_tiles = w.p_tiles * w.q_tiles;
  const int first = (int)(blockIdx.x >> 1), stride = (int)(gridDim.x >> 1);
  // the other CTA learns of a wait that gave up
  auto give_up = [&]() {
    abort_flag = 1;
    const uint32_t other = map_to(smem_u32(&abort_flag), rank ^ 1u);
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(other), "r"(1u) : "memory");
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      if (s % 2 == 0) mbar_init(&full[s / 2], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SF_SLOTS; ++s) {
      mbar_init(&sf_full[s], 2);
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(&acc_empty[0], 2 * C::EPI);
    mbar_init(&acc_empty[1], 2 * C::EPI);
    mbar_init(&drain, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  after_earlier_kernels();
  // through a warp reduction: it lands in a uniform register, where the MMAs want it
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, tmem_base);

  if (warp == 0) {
    const bool one = elect_one();
    Ring<C::STAGES / 2> st;
    Fills fills[2];   // of the slots' first and second blocks
    bool ok = true;
    for (int t = first; t < n_tiles && ok; t += stride) {
      int64_t p0, q0;
      pair_origin(t, w, BN, p0, q0);
      p0 += rank * BM;
      q0 += rank * (BN / 2);
      for (int kb = 0; kb < g.kblocks && ok; kb += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // an odd last block leaves the second slot of its two empty
          const bool used = kb + h < g.kblocks;
          if (used && ok && fills[h].any(st.slot)) ok = wait_warp(&empty[2 * st.slot + h], fills[h].latest(st.slot), abort_v);
          if (used && ok) {
            if (one) {
              unsigned char* sp = smem + (2 * st.slot + h) * C::STAGE_BYTES;
              const uint32_t bar = map_to(smem_u32(&full[st.slot]), 0);
              if (rank == 0 && h == 0) mbar_arrive_tx(&full[st.slot], kb + 1 < g.kblocks ? 4 * C::STAGE_BYTES : 2 * C::STAGE_BYTES);
              tma_load_pair(sp, &map_p, (kb + h) * BK, (int)p0, bar);
              tma_load_pair(sp + C::A_BYTES, &map_q, (kb + h) * BK, (int)q0, bar);
            }
            __syncwarp();
            fills[h].next(st.slot);
          }
        }
        if (!ok) give_up();
        st.next();
      }
    }
    // the even CTA's commits arrive here too: its last ones have come before
    // this CTA's shared memory goes to another
    for (int s = 0; s < C::STAGES && ok; ++s)
      if (fills[s & 1].any(s >> 1)) ok = wait_warp(&empty[s], fills[s & 1].latest(s >> 1), abort_v);
    if (!ok) give_up();
    // both CTAs' loads report to the even one's barriers, where they are awaited should a wait have given up
    if (one)
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(map_to(smem_u32(loads[rank]), 0)), "r"(fills[0].begun),
                   "r"(fills[0].parity)
                   : "memory");
  } else if (warp == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      const uint32_t tiles_lo = desc_lo(smem_u32(smem)), sf_lo = desc_lo(smem_u32(smem + C::SF_OFF));
      const uint32_t idesc = instr_desc(2 * BM, BN, g.p.code, g.q.code);
      Ring<C::STAGES / 2> st;
      Ring<SF_SLOTS> sf, freed;   // freed: the group whose MMAs must be done before a scale buffer is written again
      Ring<C::SF_BUFS> buf;
      uint32_t item = 0, groups = 0;
      bool ok = true;
      for (int t = first; t < n_tiles && ok; t += stride) {
        for (int ch = 0; ch < w.chunks && ok; ++ch, ++item) {
          const int kb0 = ch * w.chunk_blocks, kb1 = min(g.kblocks, kb0 + w.chunk_blocks);
          if (C::SHARED) {
            if (item > 0) ok = wait_warp(&acc_empty[0], (item - 1) & 1u, abort_v);
          } else if (item > 1) {
            ok = wait_warp(&acc_empty[item & 1u], (item / 2 - 1) & 1u, abort_v);
          }
          const uint32_t acc = tmem + (item & 1u) * C::ACC_STRIDE;
          for (int kb = kb0; kb < kb1 && ok; kb += 4, ++groups) {
            const uint32_t sfp = tmem + C::SF_COL + buf.slot * C::SF_COLS, sfq = sfp + 4;
            ok = wait_warp(&sf_full[sf.slot], sf.phase, abort_v);
            if (ok && groups >= C::SF_BUFS) {
              ok = wait_warp(&sf_empty[freed.slot], freed.phase, abort_v);
              freed.next();
            }
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = sf_lo + sf.slot * (SF_SLOT_BYTES / 16);
            copy_scales_pair(sfp, desc_at(src, SCALE_HI), one);
            copy_scales_pair(sfq, desc_at(src + 32, SCALE_HI), one);
            if (BN > 128) copy_scales_pair(sfq + 4, desc_at(src + 64, SCALE_HI), one);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              if (kb + j < kb1 && ok) {
                ok = wait_warp(&full[st.slot], st.phase, abort_v);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  if (kb + j + h < kb1) {
                    const uint32_t lo = tiles_lo + (2 * st.slot + h) * (C::STAGE_BYTES / 16);
                    mma_block<true>(acc, lo, lo + C::A_BYTES / 16, idesc | sf_id(j + h), sfp, sfq, kb + j + h > kb0,
                                    &empty[2 * st.slot + h], TILE_HI, one);
                  }
                }
                st.next();
              }
            }
            commit_pair(&sf_empty[sf.slot], one);
            sf.next();
            buf.next();
          }
          if (ok) commit_pair(&acc_full[item & 1u], one);
        }
      }
      if (!ok) give_up();
    }
  } else if (warp < 4) {
    // warps 2 and 3 take the groups in turn, each loading its next one before
    // it stores the present one: one warp that loaded and stored in turn took
    // 2500 cycles for a group whose MMAs take 2048
    const int per_tile = (g.kblocks + 3) / 4;
    const int n_groups = (n_tiles - first + stride - 1) / stride * per_tile;   // first < n_tiles: the grid is no larger
    ScaleWords<BN> now, then;
    auto load = [&](ScaleWords<BN>& w4, int i) {
      int64_t p0, q0;
      pair_origin(first + i / per_tile * stride, w, BN, p0, q0);
      w4.load(g, p0 + rank * BM, q0, i % per_tile, lane);
    };
    int i = warp - 2;
    bool ok = true;
    if (i < n_groups) load(now, i);
    for (; i < n_groups; i += 2) {
      const int slot = i % SF_SLOTS;
      if (i + 2 < n_groups) load(then, i + 2);
      if (i >= SF_SLOTS) ok = wait_warp(&sf_empty[slot], (uint32_t)(i / SF_SLOTS - 1) & 1u, abort_v);
      if (!ok) {
        if (lane == 0) give_up();
        break;
      }
      now.store(smem + C::SF_OFF + slot * SF_SLOT_BYTES, lane);
      __syncwarp();
      if (lane == 0) arrive_at(map_to(smem_u32(&sf_full[slot]), 0));
      now = then;
    }
    for (int j = n_groups > SF_SLOTS ? n_groups - SF_SLOTS : 0; j < n_groups && ok; ++j)
      ok = wait_warp(&sf_empty[j % SF_SLOTS], (uint32_t)(j / SF_SLOTS) & 1u, abort_v);
    if (!ok && lane == 0) give_up();
  } else if (warp >= 4) {
    const uint32_t step = g.drop ? drop_step(d) : 0u;
    const int quarter = warp & 3, share = (warp - 4) >> 2;
    unsigned char* turn = smem + C::TURN_OFF + (warp - 4) * 4096;
    const uint32_t empty_bar[2] = {map_to(smem_u32(&acc_empty[0]), 0), map_to(smem_u32(&acc_empty[1]), 0)};
    uint32_t item = 0;
    bool ok = true;
    for (int t = first; t < n_tiles && ok; t += stride) {
      int64_t p0, q0;
      pair_origin(t, w, BN, p0, q0);
      const int64_t p = p0 + rank * BM + quarter * 32;
      for (int ch = 0; ch < w.chunks; ++ch, ++item) {
        const uint32_t odd = item & 1u;
        ok = wait_warp(&acc_full[odd], (item >> 1) & 1u, abort_v);
        if (!ok) {
          if (lane == 0) give_up();
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + odd * C::ACC_STRIDE;
        // this warp's blocks: every EPI / 4-th of the tile's.  The columns shared
        // with the other accumulator come first.
        constexpr int BLOCKS = BN / 32, SHARE = C::EPI / 4;
        const int mine = (BLOCKS - share + SHARE - 1) / SHARE;
        auto column = [&](int i) {
          const int b = share + i * SHARE;
          return 32 * (C::SHARED && !odd ? (b == 0 ? BLOCKS - 1 : b - 1) : b);
        };
        auto release = [&]() {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_at(empty_bar[C::SHARED ? 0 : odd]);
        };
        uint32_t r[32];
        tmem_ld32(taddr + column(0), r);
        tmem_wait32(r);
        if (C::SHARED || mine == 1) release();
        // one copy of the loop's body: unrolled, it ran into instruction cache misses
#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
          turn_in(turn, r);
          if (i + 1 < mine) tmem_ld32(taddr + column(i + 1), r);   // on its way while this block goes out
          emit_block<BF16, EXTRA>(g, d, step, turn, p, q0 + column(i), ch > 0, ch == w.chunks - 1);
          if (i + 1 < mine) {
            tmem_wait32(r);
            if (!C::SHARED && i + 2 == mine) release();
          }
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  if (abort_flag) {
    // wait (bounded) for the MMAs in flight (the thread that issued them) and for loads to land
    if (warp == 1 && rank == 0 && elect_one()) {
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&drain))
                   : "memory");
      mbar_wait(&drain, 0, 1u << 20);
    }
    if (threadIdx.x == 0) {
      if (rank == 0) {
        // One CTA may have got a fill further than the other.  Its phase, or that of the fill which the other
        // has no part in, does not end then: the wait's limit is what gives the loads the time to land.
        for (int r = 0; r < 2; ++r)
          await_fills(Fills{loads[r][0], loads[r][1]}, C::STAGES / 2,
                      [&](int slot, uint32_t parity) { mbar_wait(&full[slot], parity, 1u << 20); });
      }
      if (g.err) *reinterpret_cast<volatile int32_t*>(g.err) = 1;
    }
    __syncthreads();
    cluster_sync();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- host ----
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

int encode_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (!g_encode) return set_error(ADVOPT_E_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  if (g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: cuTensorMapEncodeTiled rejected an operand");
  return ADVOPT_OK;
}

// A kernel's shared-memory limit, raised once for each device (`ready`: a bit a device).
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (ready.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  return e;
}

struct Launch {
  const void *p, *q;
  int64_t ldp, ldq, k;
  GemmArgs g;
  DropSpec d;
  cudaStream_t stream;
};

template <int BN, int S, bool BF16, bool LONG>
int launch_t(const Launch& L) {
  using C = Cfg<BN, LONG>;
  CUtensorMap mp, mq;
  int rc = encode_map(&mp, L.p, L.g.p.extent, L.k, L.ldp, BM);
  if (rc == ADVOPT_OK) rc = encode_map(&mq, L.q, L.g.q.extent, L.k, L.ldq, BN);
  if (rc != ADVOPT_OK) return rc;
  const auto kernel = gemm_kernel<BN, S, BF16, LONG>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(kernel, C::SMEM, ready);
  if (e != cudaSuccess) return check_cuda(e, "advopt_fp8_gemm: smem attribute");
  const int64_t tiles = ((L.g.p.extent + BM - 1) / BM) * ((L.g.q.extent + BN - 1) / BN);
  if (tiles * S > 0x7fffffff) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_gemm: too many output tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = L.stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = S;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kernel, mp, mq, L.g, L.d);
  return check_cuda(e, "advopt_fp8_gemm");
}

template <int BN, bool BF16>
int launch_pair(const Launch& L) {
  using C = PairCfg<BN>;
  CUtensorMap mp, mq;
  int rc = encode_map(&mp, L.p, L.g.p.extent, L.k, L.ldp, BM);
  if (rc == ADVOPT_OK) rc = encode_map(&mq, L.q, L.g.q.extent, L.k, L.ldq, BN / 2);
  if (rc != ADVOPT_OK) return rc;
  const bool extra = L.g.bias || L.g.residual || L.g.drop;
  const auto kernel = extra ? pair_kernel<BN, BF16, true> : pair_kernel<BN, BF16, false>;
  static std::atomic<uint64_t> ready[2];
  cudaError_t e = allow_smem(kernel, C::SMEM, ready[extra]);
  if (e != cudaSuccess) return check_cuda(e, "advopt_fp8_gemm: smem attribute");
  PairArgs w;
  w.p_tiles = (int)((L.g.p.extent + 2 * BM - 1) / (2 * BM));
  w.q_tiles = (int)((L.g.q.extent + BN - 1) / BN);
  // the kernel counts a pair's tiles and scale groups in 32 bits
  if ((int64_t)w.p_tiles * w.q_tiles > (1 << 30) ||
      ((int64_t)w.p_tiles * w.q_tiles / PAIRS + 1) * ((L.g.kblocks + 3) / 4) > (1 << 30))
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_gemm: too many output tiles");
  w.band = 8;
  while (w.band < 32 && (2.0 * w.band * 2 * BM + (double)PAIRS / (2 * w.band) * BN) * (double)L.k <= 40e6) w.band *= 2;
  w.chunks = BF16 ? 1 : (L.g.kblocks + CHUNK - 1) / CHUNK;
  w.chunk_blocks = ((L.g.kblocks + w.chunks - 1) / w.chunks + 3) / 4 * 4;
  w.chunks = (L.g.kblocks + w.chunk_blocks - 1) / w.chunk_blocks;
  const int tiles = w.p_tiles * w.q_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < PAIRS ? tiles : PAIRS)));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = L.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, mp, mq, L.g, w, L.d);
  return check_cuda(e, "advopt_fp8_gemm");
}

template <int BN, bool BF16, bool LONG>
int launch_s(const Launch& L, int split) {
  switch (split) {
    case 8: return launch_t<BN, 8, BF16, LONG>(L);
    case 4: return launch_t<BN, 4, BF16, LONG>(L);
    case 2: return launch_t<BN, 2, BF16, LONG>(L);
    default: return launch_t<BN, 1, BF16, LONG>(L);
  }
}

template <bool BF16, bool LONG>
int launch_n(const Launch& L, int bn, int split) {
  switch (bn) {
    case 32: return launch_s<32, BF16, LONG>(L, split);
    case 64: return launch_s<64, BF16, LONG>(L, split);
    case 128: return launch_s<128, BF16, LONG>(L, split);
    default: return launch_s<256, BF16, LONG>(L, split);
  }
}

// Which kernel, tile and split a shape gets: the least of an estimate in
// microseconds whose constants come from timing every variant on about forty
// shapes of 1 x 1024 .. 8192 x 14336 x 14336 on one B200 (back to back calls,
// cold operands).  Over those shapes the variant it picks is within 5% of the
// fastest one (geometric mean).  What it weighs:
//   * pairs (256 x BN tiles): a K block costs the MMAs' 2 BN cycles, more below
//     BN = 256 where the staged bytes per MMA grow (475 / 440 / 400); BN = 256
//     waits 2800 cycles between tiles for the shared accumulator columns, so
//     8192 x 14336 x 4096 takes 336 us at 256 and 322 at 224, and
//     8192 x 4096 x 14336 324 and 359;
//   * single CTAs (128 x BN): a K block costs what 16 KB + BN * 128 bytes take
//     from L2 (170 .. 680 cycles); splitting K pays a cluster's exchange:
//     1 x 4096 x 4096 takes 10.9 / 8.5 / 7.4 / 6.9 us split 1 / 2 / 4 / 8,
//     256 x 4096 x 4096 at BN = 64 10.5 us unsplit, at BN = 128 11.0 split in 2;
//   * a float32 sum that takes a CTA's accumulators several times over takes
//     another launch each time, 6.5 us of a single wave: 256 x 256 x 262144 split
//     in 8 takes 58 us at BN = 64 in one launch, 72 at BN = 128 in two; and more of
//     several: 1024 x 1024 x 131072 at BN = 256 takes 211 us split in 8 (two waves,
//     two launches), 148 split in 4 (one wave, four launches), 375 in pairs;
//   * swapped operands write D a token at a time, a feature per lane, whatever
//     D's alignment: 333 x 2041 x 1000 takes 5.3 us swapped, 6.1 not.
struct Variant {
  bool pair, swap;
  int bn, split;
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline Variant choose(int64_t m, int64_t n, int64_t kblocks, bool whole_rows, bool f32) {
  Variant best{false, false, 32, 1};
  double least = 1e300;
  static constexpr int single_bn[4] = {32, 64, 128, 256}, pair_bn[4] = {256, 224, 192, 128};
  static constexpr double single_block[4] = {330, 340, 440, 680}, pair_block[4] = {512, 475, 440, 400};
  static constexpr double pair_gap[4] = {2800, 400, 400, 400}, pair_out[4] = {10000, 8500, 7500, 5500};
  for (int swap = 0; swap < 2; ++swap) {
    const int64_t p = swap ? n : m, q = swap ? m : n;
    for (int lg = 0; lg < 4; ++lg) {
      const int split = 1 << lg;
      if (split > 1 && ceil_div(kblocks, 4) < split) break;
      for (int i = 0; i < 4; ++i) {
        const int bn = single_bn[i];
        if (i > 0 && bn >= 2 * q) break;
        const double ctas = (double)ceil_div(p, 128) * ceil_div(q, bn) * split;
        const double waves = ceil_div((int64_t)ctas, i == 0 ? 2 * SMS : SMS);   // BN = 32: two CTAs fit an SM
        double block = single_block[i];
        if (i == 0) block = ctas > SMS ? 400 : ctas * 330 / SMS > 170 ? ctas * 330 / SMS : 170;
        if (i == 0 && q > 32) block *= 1.4;   // the other operand is read again for each 32 columns
        const int64_t groups = ceil_div(kblocks, 4), sums = split * (CHUNK / 4);
        const int64_t parts = f32 ? ceil_div(groups, sums * long_accs(bn)) : 1;
        if (f32 && groups > sums && split < 8 && kblocks <= 8 * CHUNK && groups >= 2 * split) continue;   // one sum a CTA
        const int64_t blocks = 4 * ceil_div(groups, split);
        const double body = (double)(blocks < kblocks ? blocks : kblocks) * block / 1800;
        const double out = bn / 32 * (swap ? 0.35 : whole_rows ? 0.3 : 0.8) / split;
        const double join = split == 1 ? 0 : bn / 32 * 0.3 + (split == 2 ? (i ? 1.0 : 0.7) : split == 4 ? 1.2 : i ? 6.0 : 1.3);
        const double t = 2.8 + (waves - 1) * (body + out + 1.2) + body + out + join + (parts - 1) * (waves > 1 ? 30.0 : 6.5);
        if (t < least) {
          least = t;
          best = Variant{false, swap != 0, bn, split};
        }
      }
    }
  }
  for (int i = 0; i < 4; ++i) {
    const double waves = (double)ceil_div(ceil_div(m, 256) * ceil_div(n, pair_bn[i]), PAIRS);
    const double tile = (double)kblocks * pair_block[i] + pair_gap[i];
    const double t = 4.0 + (waves * (tile > 0.7 * pair_out[i] ? tile : 0.7 * pair_out[i]) + 0.8 * pair_out[i]) / 1750;
    if (t < least) {
      least = t;
      best = Variant{true, false, pair_bn[i], 1};
    }
  }
  return best;
}

// advopt_fp8_gemm_args.variant: BN of a pair kernel, or 1000 * split + BN of a
// single-CTA kernel, plus 100000 with the operands swapped.
inline bool named(int32_t code, int64_t groups, Variant* v) {
  if (code < 0) return false;
  const int swap = code / 100000, split = code % 100000 / 1000, bn = code % 1000;
  *v = Variant{split == 0, swap == 1, bn, split ? split : 1};
  if (swap > 1) return false;
  if (v->pair) return !swap && (bn == 128 || bn == 192 || bn == 224 || bn == 256);
  return (bn == 32 || bn == 64 || bn == 128 || bn == 256) && (split == 1 || split == 2 || split == 4 || split == 8) &&
         split <= groups;
}

}  // namespace fp8
}  // namespace advopt

using namespace advopt;

extern "C" int advopt_fp8_gemm(const advopt_fp8_gemm_args* a, void* stream) {
  if (!a || a->m < 0 || a->n < 0 || a->k <= 0) return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: bad shape");
  if (a->d_dtype != ADVOPT_DT_F32 && a->d_dtype != ADVOPT_DT_BF16)
    return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_gemm: float32 and bfloat16 outputs are supported");
  if ((a->a_code & ~1) || (a->b_code & ~1)) return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: unknown code type");
  if (const char* why = drop_check(a->drop)) return set_error(ADVOPT_E_INVALID, why);
  if (a->m == 0 || a->n == 0) return ADVOPT_OK;
  if (!a->a || !a->b || !a->sa || !a->sb || !a->d) return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: null operand");
  if ((reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->b)) % 16 || a->lda % 16 || a->ldb % 16 ||
      a->lda < a->k || a->ldb < a->k)
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: operands must be 16-byte aligned with pitches of whole 16 bytes");
  const int64_t nb = (a->k + 127) / 128;
  if ((reinterpret_cast<uintptr_t>(a->sa) | reinterpret_cast<uintptr_t>(a->sb)) % 4 || a->ldsa % 4 || a->ldsb % 4 ||
      a->ldsa < nb || a->ldsb < nb)
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: scales must be 4-byte aligned with pitches of whole 4 bytes");
  if (a->ldd < a->n || (a->residual && a->ldres < a->n))
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: a row pitch is smaller than a row");
  const int64_t top = 0x7fffff00;
  if (a->m > top || a->n > top || a->k > top) return set_error(ADVOPT_E_UNSUPPORTED, "advopt_fp8_gemm: extents are at most 2^31 - 256");

  fp8::Launch L;
  const fp8::Side A{a->sa, a->ldsa, a->m, a->a_tile ? 7 : 0, a->a_code};
  const fp8::Side B{a->sb, a->ldsb, a->n, a->b_tile ? 7 : 0, a->b_code};
  const bool bf16 = a->d_dtype == ADVOPT_DT_BF16;
  fp8::Variant v = fp8::choose(a->m, a->n, nb, a->n * (bf16 ? 2 : 4) % 16 == 0, !bf16);
  if (a->variant && !fp8::named(a->variant, (nb + 3) / 4, &v))
    return set_error(ADVOPT_E_INVALID, "advopt_fp8_gemm: no such variant for this shape");
  const bool swap = v.swap;
  fp8::GemmArgs& g = L.g;
  g.p = swap ? B : A;
  g.q = swap ? A : B;
  L.p = swap ? a->b : a->a;
  L.q = swap ? a->a : a->b;
  L.ldp = swap ? a->ldb : a->lda;
  L.ldq = swap ? a->lda : a->ldb;
  L.k = a->k;
  g.d = a->d;
  g.bias = a->bias;
  g.residual = a->residual;
  g.ldd = a->ldd;
  g.ldres = a->ldres;
  g.n = a->n;
  g.kblocks = (int)nb;
  g.swap = swap;
  const int64_t es = a->d_dtype == ADVOPT_DT_BF16 ? 2 : 4;
  g.vec = reinterpret_cast<uintptr_t>(a->d) % 16 == 0 && a->ldd * es % 16 == 0 &&
          (!a->residual || (reinterpret_cast<uintptr_t>(a->residual) % 16 == 0 && a->ldres * es % 16 == 0));
  g.vec_bias = reinterpret_cast<uintptr_t>(a->bias) % 16 == 0;
  g.drop = a->drop.threshold > 0;
  g.more = 0;
  g.err = a->err;
  L.d = drop_spec(a->drop);
  L.stream = static_cast<cudaStream_t>(stream);
  if (v.pair) {
    switch (v.bn) {
      case 256: return bf16 ? fp8::launch_pair<256, true>(L) : fp8::launch_pair<256, false>(L);
      case 224: return bf16 ? fp8::launch_pair<224, true>(L) : fp8::launch_pair<224, false>(L);
      case 192: return bf16 ? fp8::launch_pair<192, true>(L) : fp8::launch_pair<192, false>(L);
      default: return bf16 ? fp8::launch_pair<128, true>(L) : fp8::launch_pair<128, false>(L);
    }
  }
  // launches, of whole scale words of K
  const int64_t groups = (nb + 3) / 4, sums = v.split * (fp8::CHUNK / 4);
  const bool longer = !bf16 && groups > sums;
  const int64_t parts = longer ? fp8::ceil_div(groups, sums * fp8::long_accs(v.bn)) : 1;
  const fp8::Launch whole = L;
  for (int64_t i = 0; i < parts; ++i) {
    const int64_t g0 = groups * i / parts, g1 = groups * (i + 1) / parts, k0 = g0 * 512;
    const bool last = i + 1 == parts;
    L.p = static_cast<const uint8_t*>(whole.p) + k0;
    L.q = static_cast<const uint8_t*>(whole.q) + k0;
    L.k = (last ? a->k : g1 * 512) - k0;
    g.p.scales = whole.g.p.scales + g0 * 4;
    g.q.scales = whole.g.q.scales + g0 * 4;
    g.kblocks = (int)((last ? nb : g1 * 4) - g0 * 4);
    g.more = i > 0;
    g.bias = last ? whole.g.bias : nullptr;
    g.residual = last ? whole.g.residual : nullptr;
    g.drop = last ? whole.g.drop : 0;
    const int rc = bf16     ? fp8::launch_n<true, false>(L, v.bn, v.split)
                   : longer ? fp8::launch_n<false, true>(L, v.bn, v.split)
                            : fp8::launch_n<false, false>(L, v.bn, v.split);
    if (rc != ADVOPT_OK) return rc;
  }
  return ADVOPT_OK;
}
