// Products of MXFP4 operands (e2m1, one e8m0 scale per 32) for any number of
// tokens, of one weight matrix or of one per expert:
//
//   y[r, n] = sum_k (a sa)[r, k] (b[e(r)] sb[e(r)])[n, k]               r: rows sorted by expert
//   gated:    silu(a . b1^T) * (a . b2^T), which may leave as MXFP4
//
// fp32 sums in the tensor cores, rounded once to the output's type.
//
// The weights' rows take the M side of the tcgen05 tile and the tokens the N
// side: M is 128 whatever the problem, while N goes down to the tokens that are
// there (in steps of 32), so a decoding step pays for its few tokens and a
// weight is never padded by more than a tile at the end of N.  Tiles of up to
// `tn` tokens are cut within each expert's rows; a TMA box that reaches past an
// expert's last row reads the next one's, whose products are not stored.
// A gated tile is 64 rows of b1 over 64 rows of b2, so that both products of
// an output share a tile, its token operand and its accumulator.
//
// One persistent CTA per SM, 21 warps:
//   0, 10..12      TMA producers (K tiles of 256 dealt round-robin)
//   1              TMEM owner, MMA issuer: tcgen05.mma kind::mxf4 block32, K = 64
//   2..5, 13..16   epilogue: two groups of four, alternate steps of 32 tokens
//   6..9, 17..20   scale writers, for the even and the odd stages: each tile's
//                  128x4 scale blocks from shared memory to TMEM (tcgen05.st;
//                  tcgen05.cp would take tensor-pipe time).  A token tile that
//                  begins inside a block of 128 takes its words from the block's
//                  middle on.
// Tiles of 128 to 256 tokens may be shared by a pair of CTAs (cta_group::2): 256
// weight rows, each CTA with its own half of them and of the tokens, which halves the
// token bytes per SM.  choose_shape weighs them with the tiles of one CTA.
//
// What bounds it, on B200: few tokens by HBM -- 32 tokens over 64 experts, gated,
// 2048x4096: 76 us for 0.56 GB, 7.4 TB/s, above the 6.6 TB/s of a copy; one token
// through 7168x16384 15.2 us, 9.5 of them traffic, the rest set-up, the first
// loads' latency and the exchange of partial sums.  Many tokens by nothing alone:
// 8192x7168x4096 (93 us, 5.1 PFLOP/s) has the tensor pipe busy for 74 % of the time,
// takes 55 bytes a clock and SM from L2 (12.9 TB/s, 43 % of what the counter has as
// its peak) and has the clock down to 1.57 GHz.  What a tile costs beside its K tiles
// (kShapes) is 22 % of it at K = 4096; 8192x7168x16384 takes 327 us (5.9 PFLOP/s, 0.88
// of 4 x the measured bf16 rate).  1000x7168x16384 (47 us, 5.0 PFLOP/s) has 112 tiles
// for 74 pairs.  Over seconds the power cap takes 15 % of these.
// The offsets are read on the device: every CTA builds the table of the experts'
// rows, scale blocks and tiles in shared memory and walks the same tile list, so
// the host never waits for a routing.
//
// Few tiles (a decoding step of one matrix): a cluster splits K and adds its
// partial sums through distributed shared memory, in rank order.
//
// Every wait is bounded.  A role whose wait runs out records it and stops; the
// others then run out of what it would have given them, within a second each.  (A
// flag that all of them read at every K tile cost 2 %.)
#include <cuda_bf16.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kernels.h"
#include "mx.cuh"

namespace nvfp4 {

bool make_tma_3d_u8(CUtensorMap* map, const void* base, uint64_t inner, uint64_t rows, uint64_t L, uint64_t row_stride,
                    uint64_t lstride, uint32_t box_inner, uint32_t box_rows);

namespace {

constexpr int kBM = 128;                 // weight rows per tile
constexpr int kBK = 256;                 // K elements per stage: 128 bytes per row
constexpr int kBKBytes = kBK / 2;
constexpr int kABytes = kBM * kBKBytes;  // weight bytes per stage
constexpr int kSfBytes = 1024;           // scales of 128 rows of one stage: two 512-byte blocks
constexpr int kMaxProducers = 4;
constexpr int kThreads = 672;
constexpr int kGroups = 2;               // epilogue groups of four warps
constexpr int kMaxStages = 10;
constexpr int kTmemCols = 512;
constexpr int kChunk = 32;               // tokens per epilogue step
constexpr int kSmallBox = 32;            // token rows of a small TMA box
constexpr int kSmemMax = 227 * 1024;

struct Params {
  const uint8_t* sfw;   // scales of the weights (b, b1)
  const uint8_t* sfw2;  // of b2 (gated)
  const uint8_t* sfx;   // scales of the tokens
  void* c;
  uint8_t* c_scales;   // Codes: the result's scales (c: its codes)
  const int* offsets;  // null: one expert with all rows
  int rows, N, K, experts;
  int64_t ldc;
  int tn;         // tokens per tile: 32, 64, 128, 192 or 256
  int nblk;       // 128-row scale blocks that a token tile can touch
  int stages, producers, acc_bufs;
  int x_cols;     // TMEM columns of the token scales of 128 K columns
  int sf_cols;    // TMEM columns of scales per stage
  int n_tiles;    // tiles along N
  int splits;     // CTAs of a cluster that share a tile's K (kSplitK)
  int pair;       // kPairs
  int vec;        // 16-byte stores of C
  int tma;        // TMA stores of C
  int* status;
  int inject;     // test hook: CTA 0 withholds its first weight load
};

// The type of a result that is quantised to MXFP4 on its way out.
struct Codes {
  uint8_t pair;
};

// How CTAs share the tiles: one each; K split over a cluster; two CTAs a tile.
enum Mode { kWhole, kSplitK, kPairs };

// D (+)= (A x sfA) (B x sfB)^T, e2m1 operands, e8m0 scales, one per 32; kTwo:
// of a pair of CTAs (M = 256, each CTA's rows of A and half of B's).
template <bool kTwo>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if (kTwo)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}

// Instruction descriptor for kind::mxf4: e2m1 operands, e8m0 scales (bit 23);
// of the four scale bytes in a TMEM word an MMA of K = 64 takes two, from byte
// 0 or 2 (scale ids, bits 4-5 for B and 29-30 for A).
__device__ __forceinline__ uint32_t idesc_mxf4(int m, int n, uint32_t scale_id) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 4) << 24) | (scale_id << 4) | (scale_id << 29);
}

// 16 lanes x 8 (32) columns in the layout of an MMA's accumulator: thread t gets
// of each 8 columns (lane t / 4, columns 2 (t % 4), + 1) and the same of lane
// t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x256b_x1(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// kN 8x8 matrices of 16-bit values, stored transposed: lane l gives the address
// of row l % 8 of matrix l / 8.
template <int kN>
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, const uint32_t* v) {
  if constexpr (kN == 4)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
  else
    asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(v[0]), "r"(v[1])
                 : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// AND of `pred` over the 128 threads of an epilogue group.
__device__ __forceinline__ bool group_all(int id, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %2, 0;\n\t"
      "bar.red.and.pred p, %1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(out)
      : "r"(id), "r"(static_cast<uint32_t>(pred))
      : "memory");
  return out != 0;
}

__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[8], const uint32_t (&s)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(s[0]), "r"(s[1]),
      "r"(s[2]), "r"(s[3]), "r"(s[4]), "r"(s[5]), "r"(s[6]), "r"(s[7])
      : "memory");
}
__device__ __forceinline__ void put4(uint32_t* dst, const uint8_t* src) {
  const uint4 v = *reinterpret_cast<const uint4*>(src);
  dst[0] = v.x;
  dst[1] = v.y;
  dst[2] = v.z;
  dst[3] = v.w;
}

// Shared-memory operands by address (uniform over the warp).
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load_u32(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}
template <bool kTwo>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z,
                                          uint64_t policy) {
  if (kTwo)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
}

// One lane of a converged warp, the same on every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// 16 bytes to another CTA's shared memory, counted on that CTA's barrier.
__device__ __forceinline__ void st_async_v4(uint32_t addr, const uint32_t* v, uint32_t bar) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar)
      : "memory");
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ __half round_to<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float round_to<float>(float v) {
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t round_pair(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The experts' rows, scale blocks and tiles, in shared memory: E + 1 ints each.
struct Table {
  const int *row, *blk, *tile;
};

struct Tile {
  int e;       // expert
  int row0;    // first row
  int rows;    // rows of the tile, 1 .. tn
  int in_blk;  // row0's place in its scale block, a multiple of 32
  int blk;     // its scale block
  int ft;      // tile along N
};

// The tile in values that the compiler knows to be the same in every lane.
__device__ __forceinline__ Tile uniform(const Tile& o) {
  return Tile{__shfl_sync(0xffffffffu, o.e, 0),      __shfl_sync(0xffffffffu, o.row0, 0),
              __shfl_sync(0xffffffffu, o.rows, 0),   __shfl_sync(0xffffffffu, o.in_blk, 0),
              __shfl_sync(0xffffffffu, o.blk, 0),    __shfl_sync(0xffffffffu, o.ft, 0)};
}

// Tile t (< tab.tile[E]); `e` is the walker's cursor.  Tiles of an expert go
// over up to kGroup token tiles for each weight tile, so that CTAs that run
// together share both operands in L2 (24 against 12: 8192x7168x4096 100 -> 98 us).
constexpr int kGroup = 24;
__device__ __forceinline__ Tile tile_at(const Params& p, const Table& tab, int t, int& e) {
  while (t >= tab.tile[e + 1]) ++e;
  const int count = tab.row[e + 1] - tab.row[e];
  const int mt = (count + p.tn - 1) / p.tn;
  int r = t - tab.tile[e];
  const int g = r / (kGroup * p.n_tiles);
  const int gm = min(mt - g * kGroup, kGroup);
  r -= g * kGroup * p.n_tiles;
  Tile o;
  o.e = e;
  o.ft = r / gm;
  const int m0 = (g * kGroup + r - o.ft * gm) * p.tn;
  o.row0 = tab.row[e] + m0;
  o.rows = min(p.tn, count - m0);
  o.in_blk = m0 & 127;
  o.blk = tab.blk[e] + (m0 >> 7);
  return o;
}

// The epilogue's staging of 32 tokens: boxes of 32 x 128 bytes with the 128-byte
// swizzle of a TMA store, so that matrices of 8 tokens x 16 bytes and whole rows
// are both free of bank conflicts.  Byte offset of feature f of token t:
template <typename OutT>
__device__ __forceinline__ int staged(int t, int f) {
  const int b = f * static_cast<int>(sizeof(OutT));
  return (b >> 7) * (kChunk * 128) + t * 128 + ((b & 112) ^ ((t & 7) << 4)) + (b & 15);
}
// Staging buffers per group: 32-bit types have one, the others write one while
// the other is stored.
__host__ __device__ constexpr int staging_bufs(size_t out_size) { return out_size <= 2 ? 2 : 1; }

// kSplitK: groups of 8 tokens that a rank adds up, and its space for the others'
// partial sums of them: 128 rows x 8 tokens in fp32 per group and rank.
__host__ __device__ constexpr int rank_share(int groups, int splits) { return (groups + splits - 1) / splits; }
__host__ __device__ constexpr int sums_bytes(int tn, int splits) {
  return rank_share(tn / 8, splits) * (splits - 1) * 4096;
}

template <typename OutT, bool kGate, Mode kMode>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w2,
                   const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_xs,
                   const __grid_constant__ CUtensorMap tm_c, const Params p) {
  constexpr int kF = kGate ? 64 : 128;  // output features per tile
  constexpr int kSfW = kGate ? 2 : 1;   // weight scale blocks per 128 columns of K
  constexpr bool kSplit = kMode == kSplitK, kPair = kMode == kPairs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = p.stages;
  const int x_rows = kPair ? p.tn / 2 : p.tn;  // token rows of a stage
  const int stage_bytes = kABytes + x_rows * kBKBytes;
  const int sf_bytes = (kSfW + p.nblk) * kSfBytes;
  constexpr bool kCodes = std::is_same<OutT, Codes>::value;
  static_assert(!kCodes || kGate, "only gated results are quantised");
  constexpr int kBufs = staging_bufs(sizeof(OutT)), kStaged = kChunk * kF * sizeof(OutT);
  uint8_t* staging = smem + S * stage_bytes;  // per group kBufs of kStaged bytes (1024-aligned)
  uint8_t* sums = staging + kGroups * kBufs * kStaged;  // kSplit: the other ranks' partial sums
  uint8_t* sfbuf = sums + (kSplit ? sums_bytes(p.tn, p.splits) : 0);
  uint4* exch = reinterpret_cast<uint4*>(sfbuf + S * sf_bytes);  // gated, per group: 512
  uint64_t* bars = reinterpret_cast<uint64_t*>(exch + (kGate ? kGroups * 512 : 0));
  uint64_t* full = bars;
  uint64_t* empty = full + S;
  uint64_t* sf_full = empty + S;
  uint64_t* acc_full = sf_full + S;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint64_t* sums_full = drain + 1;  // kSplit: the other ranks' partial sums are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_full + 1);
  int* row_tab = reinterpret_cast<int*>(tmem_slot + 2);
  int* blk_tab = row_tab + p.experts + 1;
  int* tile_tab = blk_tab + p.experts + 1;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int KT = (p.K + kBK - 1) / kBK, K128 = (p.K + 127) >> 7;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], kPair ? 1 + 8 : 1 + 4);  // the producer, and each scale writer (of both CTAs)
      mbar_init(&empty[s], 1);
      mbar_init(&sf_full[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (kPair ? 2 : 1) * kGroups * 128);
    }
    mbar_init(drain, 1);
    mbar_init(sums_full, 1);
    fence_barrier_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    prefetch_tensormap(&tm_xs);
    if (kGate) prefetch_tensormap(&tm_w2);
    pdl_allow_dependents();
  }
  if (warp == 1) {
    if (kPair)
      tmem_alloc_pair(tmem_slot, kTmemCols);
    else
      tmem_alloc(tmem_slot, kTmemCols);
  }
  // Table of the experts, then the running number of their tiles (warp 0).
  auto build_table = [&]() {
    if (p.offsets) {
      load_expert_table(p.offsets, p.experts, p.rows, row_tab, blk_tab);
    } else if (lane == 0) {
      row_tab[0] = blk_tab[0] = 0;
      row_tab[1] = p.rows;
    }
    __syncwarp();
    int carry = 0;
    for (int base = 0; base < p.experts; base += 32) {
      const int e = base + lane;
      int n = e < p.experts ? (row_tab[e + 1] - row_tab[e] + p.tn - 1) / p.tn * p.n_tiles : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, n, d);
        if (lane >= d) n += o;
      }
      n += carry;
      if (e < p.experts) tile_tab[e + 1] = n;
      carry = __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) tile_tab[0] = 0;
  };
  // What needs nothing of the kernel before runs while that one drains.
  if (warp == 0 && !p.offsets) build_table();
  tc_fence_before();
  if (kPair || kSplit)
    cluster_sync_all();  // the other CTAs' barriers and TMEM are there
  else
    __syncthreads();
  tc_fence_after();
  pdl_wait();
  if (p.offsets) {
    if (warp == 0) build_table();
    __syncthreads();
  }
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t sf_col0 = p.acc_bufs * p.tn;
  const Table tab{row_tab, blk_tab, tile_tab};
  const int total = tile_tab[p.experts];
  // Work of this CTA: tiles t0, t0 + step, .., K tiles [k0, k1) of each.
  const int t0 = kSplit ? blockIdx.x / p.splits : kPair ? blockIdx.x >> 1 : blockIdx.x;
  const int step = kSplit ? total : kPair ? gridDim.x >> 1 : gridDim.x;  // kSplit: one tile per cluster
  const int rank = kMode == kWhole ? 0 : static_cast<int>(cluster_ctarank());
  // A tile's first scale row, of its tokens and of a quantised result.
  auto scale0 = [&](const Tile& o) { return static_cast<int64_t>(o.blk) * 128 + o.in_blk; };
  // First feature of this CTA's weight rows.
  auto feature0 = [&](const Tile& o) { return kPair ? (2 * o.ft + rank) * kF : o.ft * kF; };
  const int k0 = kSplit ? rank * KT / p.splits : 0, k1 = kSplit ? (rank + 1) * KT / p.splits : KT;
  bool partial_ready = false;  // epilogue threads, kSplit: this CTA's partial sums are in TMEM

  const int producer = warp == 0 ? 0 : warp >= 10 && warp <= 12 ? warp - 9 : -1;
  if (producer >= 0) {
    // ------------------------------------------------------------ producers
    // K tile g of this CTA's sequence (over all its tiles) goes to producer
    // g % producers, in stage g % S; counters instead of remainders, whose
    // divisions took longer than the copies.
    // (As the MMA issuer, the whole warp walks and one lane issues.)
    if (producer < p.producers) {
      const bool issue = elect_one();
      const int tiles = __shfl_sync(0xffffffffu, total, 0);
      const uint64_t keep = policy_evict_last(), once = policy_evict_first();
      const int P = p.producers;
      int e = 0, stage = producer;
      int ahead = producer;  // this producer's next K tile, counted from the tile's first
      uint32_t phase = 1;
      const int wblocks = (p.N + 127) >> 7;
      const uint32_t stages0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint32_t sf0 = __shfl_sync(0xffffffffu, smem_u32(sfbuf), 0);
      const uint32_t full0 = __shfl_sync(0xffffffffu, smem_u32(full), 0), sf_full0 = full0 + 16 * S;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step) {
        const Tile o = uniform(tile_at(p, tab, t, e));
        const int f0 = feature0(o);
        // (The second CTA's rows may all lie past N: any block's scales do.)
        const int64_t wsf = (static_cast<int64_t>(o.e) * wblocks + min(f0 >> 7, wblocks - 1)) * K128 * 512;
        const uint8_t* xsf = p.sfx + static_cast<int64_t>(o.blk) * K128 * 512;
        const int nb = ((o.in_blk + o.rows - 1) >> 7) + 1;
        // The tile's tokens, or this CTA's half of the columns that the MMA
        // takes: in one box, or in small ones where that would read much more.
        const int half = ((o.rows + 31) & ~31) >> 1;
        const int x0 = kPair ? o.row0 + rank * half : o.row0;
        const int need = kPair ? half : o.rows, small = (need + kSmallBox - 1) / kSmallBox;
        const bool one_box = 4 * need > 3 * x_rows || small == 1;
        const CUtensorMap* map_x = 4 * need > 3 * x_rows ? &tm_x : &tm_xs;
        const uint32_t box_bytes = (4 * need > 3 * x_rows ? x_rows : kSmallBox) * kBKBytes;
        const int boxes = one_box ? 1 : small;
        // A pair's loads all complete on the first CTA's barrier.
        const uint32_t tx = (kABytes + boxes * box_bytes) * (kPair ? 2 : 1);
        int kt = k0 + ahead;
        for (; kt < k1; kt += P) {
          if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase))) {
            if (issue) set_status(p.status, kStatusTimeoutEmpty);
            ok = false;
            break;
          }
          if (issue) {
            const uint32_t st = stages0 + stage * stage_bytes, sf = sf0 + stage * sf_bytes;
            const uint32_t bar = full0 + 8 * stage, sf_bar = sf_full0 + 8 * stage;
            const uint32_t bytes = min(2, K128 - 2 * kt) * 512;
            expect_tx(sf_bar, (kSfW + nb) * bytes);
            bulk_load_u32(sf, p.sfw + wsf + kt * kSfBytes, bytes, sf_bar, once);
            if (kGate) bulk_load_u32(sf + kSfBytes, p.sfw2 + wsf + kt * kSfBytes, bytes, sf_bar, once);
            bulk_load_u32(sf + kSfW * kSfBytes, xsf + 2 * kt * 512, bytes, sf_bar, keep);
            if (nb > 1)
              bulk_load_u32(sf + (kSfW + 1) * kSfBytes, xsf + (static_cast<int64_t>(K128) + 2 * kt) * 512, bytes, sf_bar,
                            keep);
            if (!kPair || rank == 0) expect_tx(bar, tx);
            const uint32_t tile_bar = kPair ? map_peer(bar, 0) : bar;
            if (!(p.inject && blockIdx.x == 0 && t == t0 && kt == k0)) {
              load_tile<kPair>(st, &tm_w, tile_bar, kt * kBKBytes, f0, o.e, once);
              if (kGate) load_tile<kPair>(st + kABytes / 2, &tm_w2, tile_bar, kt * kBKBytes, f0, o.e, once);
            }
            for (int b = 0; b < boxes; ++b)
              load_tile<kPair>(st + kABytes + b * box_bytes, map_x, tile_bar, kt * kBKBytes, x0 + b * kSmallBox, 0, keep);
          }
          __syncwarp();
          stage += P;
          if (stage >= S) {
            stage -= S;
            phase ^= 1;
          }
        }
        ahead = kt - k1;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (of a pair: the first CTA's)
    // The whole warp walks the loop and one lane issues: with every operand
    // uniform over the warp the compiler keeps the descriptors in uniform
    // registers.  (Inside a one-lane branch each tcgen05.mma cost ~125 cycles of
    // moves, 800 per K tile, more than its 4 MMAs take.)
    if (!kPair || rank == 0) {
      const bool issue = elect_one();
      const int tiles = __shfl_sync(0xffffffffu, total, 0);
      const uint64_t desc0 = desc_kmajor_sw128(__shfl_sync(0xffffffffu, smem_u32(smem), 0));
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint32_t sf0 = tmem + sf_col0;
      const int tail = (p.K - (KT - 1) * kBK + 63) >> 6;  // MMAs of the last K tile
      int stage = 0, acc = 0, e = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += step) {
        const int n = __shfl_sync(0xffffffffu, (tile_at(p, tab, t, e).rows + 31) & ~31, 0);
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], acc_phase ^ 1))) {
          if (issue) set_status(p.status, kStatusTimeoutAccEmpty);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + acc * p.tn;
        const uint32_t id0 = idesc_mxf4(kPair ? 2 * kBM : kBM, n, 0), id2 = idesc_mxf4(kPair ? 2 * kBM : kBM, n, 2);
        for (int kt = k0; kt < k1; ++kt) {
          if (!__all_sync(0xffffffffu, kPair ? mbar_wait_cluster(&full[stage], phase) : mbar_wait(&full[stage], phase))) {
            if (issue) set_status(p.status, kStatusTimeoutFull);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = desc0 + static_cast<uint32_t>(stage * stage_bytes >> 4), b = a + (kABytes >> 4);
          const uint32_t sfw = sf0 + stage * p.sf_cols, sfx = sfw + 8, more = p.x_cols;
          const int steps = kt == KT - 1 ? tail : 4;
          if (issue) {
            mma_mxf4<kPair>(d, a, b, id0, sfw, sfx, kt != k0);
            if (steps > 1) mma_mxf4<kPair>(d, a + 2, b + 2, id2, sfw, sfx, 1);
            if (steps > 2) mma_mxf4<kPair>(d, a + 4, b + 4, id0, sfw + 4, sfx + more, 1);
            if (steps > 3) mma_mxf4<kPair>(d, a + 6, b + 6, id2, sfw + 4, sfx + more, 1);
            if (kPair)
              tc_commit_pair_mc(&empty[stage], 0x3);
            else
              tc_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (issue) {
          if (kPair)
            tc_commit_pair_mc(&acc_full[acc], 0x3);
          else
            tc_commit(&acc_full[acc]);
        }
        __syncwarp();
        if (++acc == p.acc_bufs) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // Every tcgen05 operation has retired before TMEM is freed.
      if (issue) {
        if (kPair)
          tc_commit_pair(drain);
        else
          tc_commit(drain);
        mbar_wait(drain, 0);
      }
      __syncwarp();
    }
  } else if ((warp >= 6 && warp <= 9) || warp >= 17) {
    // ------------------------------------------------------------ scale writers
    // Two sets of four warps, one for the even stages and one for the odd: one
    // set's chain of wait, load, store and arrival took ~540 cycles a K tile, more
    // than the MMAs.  (By stage and not by K tile: a set waits for a stage by phase
    // parity, which is exact only if it has itself seen the stage's previous phase.
    // With sets by K tile and an odd number of stages it has seen only every other
    // one, and can take the phase before the last for its own.)  Warp i writes
    // lane quarter i % 4.  Columns of a stage: the weights' two blocks of 128 K
    // columns (4 TMEM columns each), then the tokens' (x_cols each); column c of an
    // operand holds the words of its rows 32 c .. 32 c + 31.
    const uint32_t quarter = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int set = warp >= 17 ? 1 : 0;
    int e = 0, stage = set, ahead = set;  // ahead: this set's next K tile, counted from the tile's first
    uint32_t phase = 0;
    bool ok = true;
    for (int t = t0; t < total && ok; t += step) {
      const Tile o = tile_at(p, tab, t, e);
      const int shift = o.in_blk >> 5;
      const int half = (feature0(o) & 127) >> 5;  // gated: the tile's first word in its weight blocks
      int kt = k0 + ahead;
      while (kt < k1) {
        if (!__all_sync(0xffffffffu, mbar_wait(&sf_full[stage], phase))) {
          if (lane == 0) set_status(p.status, kStatusTimeoutFull);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint8_t* sf = sfbuf + stage * sf_bytes + lane * 16;
        const uint32_t col = tmem_base + quarter + sf_col0 + stage * p.sf_cols;
        // (Blocks that were not loaded give words of columns that nobody reads.)
        uint32_t w[8], x[2][8];
        if (kGate) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint2 v = *reinterpret_cast<const uint2*>(sf + h * kSfBytes + kb * 512 + half * 4);
              w[4 * kb + 2 * h] = v.x;
              w[4 * kb + 2 * h + 1] = v.y;
            }
        } else {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) put4(w + 4 * kb, sf + kb * 512);
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          put4(x[kb], sf + kSfW * kSfBytes + kb * 512);
          if (p.nblk > 1)
            put4(x[kb] + 4, sf + (kSfW + 1) * kSfBytes + kb * 512);
          else
#pragma unroll
            for (int i = 4; i < 8; ++i) x[kb][i] = 0;
        }
        const int left = (p.K >> 5) - 8 * kt;  // scales per row from this K tile on
        if (left < 8) {
          // Padding columns are not the caller's to fill: read as 2^-127.
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const int n = left - 4 * kb;
            const uint32_t mask = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * kb + i] &= mask;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[kb][i] &= mask;
          }
        }
        if (shift & 1) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[kb][i] = i < 7 ? x[kb][i + 1] : 0;
        }
        if (shift & 2) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[kb][i] = i < 6 ? x[kb][i + 2] : 0;
        }
        if (p.x_cols == 8) {
          tmem_st_32x32b_x8(col, w);
          tmem_st_32x32b_x16(col + 8, x[0], x[1]);
        } else if (p.x_cols == 6) {
          const uint32_t some[8] = {x[0][0], x[0][1], x[0][2], x[0][3], x[0][4], x[0][5], x[1][0], x[1][1]};
          tmem_st_32x32b_x16(col, w, some);
          tmem_st_32x32b_x4(col + 16, make_uint4(x[1][2], x[1][3], x[1][4], x[1][5]));
        } else {
          const uint32_t both[8] = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
          tmem_st_32x32b_x16(col, w, both);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        // (Relaxed: the stores are complete and fenced; a release at cluster
        // scope costs over a thousand cycles.)
        if (lane == 0) {
          if (kPair)
            mbar_arrive_cluster_relaxed(map_peer(smem_u32(&full[stage]), 0));
          else
            mbar_arrive(&full[stage]);
        }
        if (stage + 2 < S) {
          stage += 2;
          kt += 2;
        } else {  // on to the set's first stage of the next lap
          kt += S - stage + set;
          stage = set;
          phase ^= 1;
        }
      }
      ahead = kt - k1;
    }
  }

  // ------------------------------------------------------------ epilogue
  const int group = warp >= 2 && warp <= 5 ? 0 : warp >= 13 && warp <= 16 ? 1 : -1;
  const int q = warp & 3;                       // lane quarter: weight rows 32 q .. 32 q + 31
  const int gtid = (warp < 6 ? warp - 2 : warp - 13) * 32 + lane;  // thread of the group
  const uint32_t tquarter = static_cast<uint32_t>(q * 32) << 16;
  OutT* const c = static_cast<OutT*>(p.c);
  // This warp's 32 weight rows x 8 G tokens in r[half][4 G] (the two halves of
  // its rows, as tcgen05.ld 16x256b leaves them) to rows row0 .. of C, features
  // f0 ..; `valid` tokens are stored.  The values pass through shared memory,
  // transposed by stmatrix so that a token's features lie together, and leave in
  // 16-byte stores.
  int buf = 0;
  auto emit = [&](auto width, uint32_t* r, int64_t row0, int64_t scale_row, int f0, int valid) {
    constexpr int G = decltype(width)::value, kR = 4 * G;
    constexpr bool kOne = kCodes && G == 1;  // the warps of x1 compute all: a block needs its 32 features in a warp
    [[maybe_unused]] constexpr int kHalves = kGate && G == 1 && !kOne ? 1 : 2;  // row halves that this warp computes
    constexpr int kTok = kGate && G > 1 ? G / 2 : G;       // its groups of 8 tokens
    uint8_t* out = staging + (group * kBufs + buf) * kStaged;
    if (kBufs == 2) {
      buf ^= 1;
    } else {  // the buffer's last store has read it
      if (gtid == 0) bulk_wait_group_read0();
      bar_sync(1 + group, 128);
    }
    int feature = q * 32, token = 0;  // of what this warp computes
    if (kOne) {
      uint4* const box = exch + group * 512 + (q & 1) * 256 + lane;
      if (q >= 2) {
        box[0] = make_uint4(r[0], r[1], r[2], r[3]);
        box[32] = make_uint4(r[4], r[5], r[6], r[7]);
      }
      bar_sync(3 + group * 2 + (q & 1), 64);
      if (q < 2) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint4 o = box[32 * v];
          const uint32_t other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            r[4 * v + i] = __float_as_uint(silu_mul(__uint_as_float(r[4 * v + i]), __uint_as_float(other[i])));
        }
      }
    } else if (kGate) {
      // Warps 0 and 1 of a group hold x1, 2 and 3 x2 of the same outputs: each
      // gives its partner half of its values (half of the tokens, or of 8 tokens
      // half of the rows) and computes the other half.
      const bool first = q < 2;
      uint4* const box = exch + group * 512 + (q & 1) * 256 + lane;
      constexpr int kV = kR / 4;  // 16-byte vectors given
      // Values given and kept, as r indices: G > 1: token groups; G == 1: row halves.
      auto at = [&](bool upper, int i) {
        return G == 1 ? (upper ? kR : 0) + i : (i / (kR / 2)) * kR + (upper ? kR / 2 : 0) + i % (kR / 2);
      };
      uint32_t keep[kR];
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        uint32_t g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i] = first ? r[at(true, 4 * v + i)] : r[at(false, 4 * v + i)];
          keep[4 * v + i] = first ? r[at(false, 4 * v + i)] : r[at(true, 4 * v + i)];
        }
        box[(first ? 0 : 128) + v * 32] = make_uint4(g[0], g[1], g[2], g[3]);
      }
      bar_sync(3 + group * 2 + (q & 1), 64);
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const uint4 o = box[(first ? 128 : 0) + v * 32];
        const uint32_t other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = __uint_as_float(first ? keep[4 * v + i] : other[i]);
          const float y = __uint_as_float(first ? other[i] : keep[4 * v + i]);
          r[4 * v + i] = __float_as_uint(silu_mul(x, y));
        }
      }
      feature = (q & 1) * 32 + (G == 1 && !first ? 16 : 0);
      token = G > 1 && !first ? 8 * kTok : 0;
    }
    // r[half][4 kTok] now, kHalves halves.
    if constexpr (kCodes) {
      // A token's 32 features of this warp are a block, four in each of the eight
      // lanes with its columns (lane / 4 + 8 k).  The scale needs only the largest
      // exponent: those of the lane's 2 kTok tokens go through three shuffles
      // together, a byte each.  Codes of neighbouring features lie in neighbouring
      // lanes (lane ^ 4), which give each other half of the tokens, so that one
      // shuffle brings whole bytes together.  They meet in shared memory: per token
      // 2 x 16 bytes of codes, then the scales.
      if (!kOne || q < 2) {
        constexpr int kT = 2 * kTok;
        const int f = lane >> 2;
        const bool odd = f & 1;
        auto value = [&](int t, int k) {
          return __uint_as_float(r[(k >> 1) * 4 * kTok + 4 * (t >> 1) + 2 * (k & 1) + (t & 1)]);
        };
        uint32_t exponents = 0;
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, __float_as_uint(value(t, k)) & 0x7fffffffu);
          exponents |= (top >> 23) << (8 * t);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) exponents = __vmaxu4(exponents, __shfl_xor_sync(0xffffffffu, exponents, d));
        uint32_t half[2] = {0, 0};  // 16 bits of codes per token
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          const uint32_t code = scale_code((exponents >> (8 * t) & 255u) << 23);
          const float inv = inverse_scale(code);
          const uint32_t n = e2m1_pair(value(t, 0) * inv, value(t, 1) * inv) |
                             e2m1_pair(value(t, 2) * inv, value(t, 3) * inv) << 8;
          half[t / kTok] |= (code == 255u ? 0u : n) << (16 * (t % kTok));
          if (f == 0)
            out[kChunk * 32 + (token + 8 * (t >> 1) + 2 * lane + (t & 1)) * 2 + (q & 1)] = static_cast<uint8_t>(code);
        }
        const uint32_t mine = odd ? half[1] : half[0];
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? half[0] : half[1], 4);
        auto spread = [](uint32_t x) {
          return (x & 0xfu) | (x & 0xf0u) << 4 | (x & 0xf00u) << 8 | (x & 0xf000u) << 12;
        };
#pragma unroll
        for (int u = 0; u < kTok; ++u) {
          const uint32_t x = spread(mine >> (16 * u)), y = spread(other >> (16 * u));
          const uint32_t bytes = odd ? y | x << 4 : x | y << 4;
          const int t = u + (odd ? kTok : 0), tok = token + 8 * (t >> 1) + 2 * (lane & 3) + (t & 1);
          uint8_t* const at = out + tok * 32 + (q & 1) * 16 + (f >> 1);
#pragma unroll
          for (int k = 0; k < 4; ++k) at[4 * k] = static_cast<uint8_t>(bytes >> (8 * k));
        }
      }
    } else if constexpr (sizeof(OutT) == 2) {
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        uint32_t m[2 * kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          m[2 * h] = round_pair<OutT>(r[h * 4 * kTok + 4 * j], r[h * 4 * kTok + 4 * j + 1]);
          m[2 * h + 1] = round_pair<OutT>(r[h * 4 * kTok + 4 * j + 2], r[h * 4 * kTok + 4 * j + 3]);
        }
        stmatrix_trans<2 * kHalves>(
            smem_u32(out + staged<OutT>(token + 8 * j + (lane & 7), feature + 8 * ((lane >> 3) & (2 * kHalves - 1)))), m);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kTok; ++j)
#pragma unroll
        for (int i = 0; i < 4 * kHalves; ++i) {
          const int h = i >> 2, f = feature + 16 * h + ((i & 2) ? 8 : 0) + (lane >> 2);
          *reinterpret_cast<OutT*>(out + staged<OutT>(token + 8 * j + 2 * (lane & 3) + (i & 1), f)) =
              round_to<OutT>(__uint_as_float(r[h * 4 * kTok + 4 * j + (i & 3)]));
        }
    }
    // A whole step, or the last rows of C, in TMA stores; the end of an expert's
    // rows, and a C whose rows do not begin and end at 16 bytes, by the threads.
    const bool tma = G == 4 && p.tma && (valid == kChunk || row0 + valid == p.rows);
    if (tma) fence_proxy_async_smem();
    if (kBufs == 2 && gtid == 0) bulk_wait_group_read0();  // the other buffer, which the next step writes, is read
    bar_sync(1 + group, 128);
    if constexpr (kCodes) {
      const int tok = (gtid & 63) >> 1, f = f0 + 32 * (gtid & 1);  // f: of the block
      if (tok < valid && f < p.N) {
        if (gtid < 64)
          *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c) + (row0 + tok) * (p.N >> 1) + (f >> 1)) =
              *reinterpret_cast<const uint4*>(out + tok * 32 + (gtid & 1) * 16);
        else
          p.c_scales[mx_scale_word(scale_row + tok, f >> 7, (p.N + 127) >> 7) + ((f >> 5) & 3)] =
              out[kChunk * 32 + tok * 2 + (gtid & 1)];
      }
    } else if (tma) {
      if (gtid == 0) {
#pragma unroll
        for (int b = 0; b < kStaged / (kChunk * 128); ++b)
          if (f0 * static_cast<int>(sizeof(OutT)) + b * 128 < p.N * static_cast<int>(sizeof(OutT)))
            tma_store_3d(&tm_c, out + b * kChunk * 128, f0 * static_cast<int>(sizeof(OutT)) + b * 128,
                         static_cast<int>(row0), 0);
        bulk_commit_group();
      }
    } else if (p.vec) {
      constexpr int kPer = 16 / sizeof(OutT), kVecs = kF / kPer;
      const int f = (gtid % kVecs) * kPer;
      if (f0 + f < p.N)  // (p.vec: N is a multiple of kPer, or ldc is more than N)
        for (int i = gtid / kVecs; i < valid; i += 128 / kVecs) {
          const uint8_t* src = out + staged<OutT>(i, f);
          OutT* dst = c + (row0 + i) * p.ldc + f0 + f;
          if (f0 + f + kPer <= p.N)
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
          else
            for (int k = 0; f0 + f + k < p.N; ++k) dst[k] = reinterpret_cast<const OutT*>(src)[k];
        }
    } else {
      for (int i = gtid; i < valid * kF; i += 128) {
        const int tok = i / kF, f = i % kF;
        if (f0 + f < p.N) c[(row0 + tok) * p.ldc + f0 + f] = *reinterpret_cast<const OutT*>(out + staged<OutT>(tok, f));
      }
    }
  };
  if (group >= 0) {
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    for (int t = t0; t < total; t += step) {
      const Tile o = tile_at(p, tab, t, e);
      // The four warps agree before any goes on to the named barriers.
      if (!group_all(1 + group, mbar_wait(&acc_full[acc], acc_phase))) {
        if (gtid == 0) set_status(p.status, kStatusTimeoutAccFull);
        break;
      }
      tc_fence_after();
      if (kSplit) {
        partial_ready = true;
        break;
      }
      const uint32_t tacc = tmem_base + tquarter + acc * p.tn;
      auto release = [&]() {
        tc_fence_before();
        if (kPair)
          mbar_arrive_cluster_relaxed(map_peer(smem_u32(&acc_empty[acc]), 0));
        else
          mbar_arrive(&acc_empty[acc]);
      };
      if (group * kChunk >= o.rows) release();
      for (int c0 = group * kChunk; c0 < o.rows; c0 += kGroups * kChunk) {
        uint32_t r[32];
        tmem_ld_16x256b_x4(tacc + c0, r);
        tmem_ld_16x256b_x4(tacc + (16u << 16) + c0, r + 16);
        tmem_wait_ld();
        if (c0 + kGroups * kChunk >= o.rows) release();
        emit(std::integral_constant<int, 4>(), r, o.row0 + c0, scale0(o) + c0, feature0(o), min(kChunk, o.rows - c0));
      }
      if (++acc == p.acc_bufs) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    // Rows that belong to no expert (their codes stay as they were).
    if constexpr (!kCodes) {
      if (group == 0) {
        const int front = row_tab[0], others = front + p.rows - row_tab[p.experts];
        for (int i = blockIdx.x; i < others; i += gridDim.x) {
          const int r = i < front ? i : row_tab[p.experts] + i - front;
          for (int f = gtid; f < p.N; f += 128) c[static_cast<int64_t>(r) * p.ldc + f] = round_to<OutT>(0.f);
        }
      }
    }
  }

  if (kSplit) {
    // ---------------------------------------------------------- partial sums of a cluster
    // Groups of 8 tokens are dealt to the ranks in contiguous shares; each rank
    // sends its partial sums of the other ranks' shares to their shared memory
    // with st.async, which counts the bytes on the receiver's barrier, and adds
    // up its own share, own sums first and then by rank: the same order always.
    // The epilogue groups take the even and the odd ones.  (With two barriers of
    // the cluster around plain stores the exchange took 2.0 us.)
    const bool ok = group >= 0 ? group_all(1 + group, partial_ready) : false;
    tc_fence_after();
    Tile o{};
    int e = 0, ng = 0;
    if (t0 < total) {
      o = tile_at(p, tab, t0, e);
      ng = (o.rows + 7) >> 3;
    }
    const int share = rank_share(ng, p.splits), first = rank * share, end = min(ng, first + share);
    if (threadIdx.x == 64) mbar_arrive_expect_tx(sums_full, max(0, end - first) * (p.splits - 1) * 4096);
    const uint32_t tacc = tmem_base + tquarter;
    auto at = [&](int slot, int gi, int half) {
      return static_cast<uint32_t>((((slot * share + gi) * 2 + half) * 128 + gtid) * 16);
    };
    if (ok) {
      constexpr int kAtOnce = 4;  // groups whose loads are in flight together
      for (int i = 1; i < p.splits; ++i) {
        const int peer = (rank + i) % p.splits;
        const uint32_t base = map_peer(smem_u32(sums), peer), bar = map_peer(smem_u32(sums_full), peer);
        const int slot = rank < peer ? rank : rank - 1;
        const int pfirst = peer * share, pend = min(ng, pfirst + share);
        for (int g0 = pfirst + ((pfirst ^ group) & 1); g0 < pend; g0 += kGroups * kAtOnce) {
          uint32_t r[kAtOnce][8];
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k)
            if (g0 + kGroups * k < pend) {
              tmem_ld_16x256b_x1(tacc + 8 * (g0 + kGroups * k), r[k]);
              tmem_ld_16x256b_x1(tacc + (16u << 16) + 8 * (g0 + kGroups * k), r[k] + 4);
            }
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k)
            if (g0 + kGroups * k < pend) {
              st_async_v4(base + at(slot, g0 + kGroups * k - pfirst, 0), r[k], bar);
              st_async_v4(base + at(slot, g0 + kGroups * k - pfirst, 1), r[k] + 4, bar);
            }
        }
      }
    }
    // No rank leaves before all have sent: whatever becomes of one rank's waits,
    // nobody writes to the shared memory of a CTA that is gone.
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (ok && !group_all(1 + group, mbar_wait_cluster(sums_full, 0))) {
      if (gtid == 0) set_status(p.status, kStatusTimeoutPeer);
    } else if (ok) {
      for (int g = first + ((first ^ group) & 1); g < end; g += kGroups) {
        uint32_t r[8];
        tmem_ld_16x256b_x1(tacc + 8 * g, r);
        tmem_ld_16x256b_x1(tacc + (16u << 16) + 8 * g, r + 4);
        tmem_wait_ld();
        for (int slot = 0; slot < p.splits - 1; ++slot)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 v = *reinterpret_cast<const float4*>(sums + at(slot, g - first, h));
            r[4 * h] = __float_as_uint(__uint_as_float(r[4 * h]) + v.x);
            r[4 * h + 1] = __float_as_uint(__uint_as_float(r[4 * h + 1]) + v.y);
            r[4 * h + 2] = __float_as_uint(__uint_as_float(r[4 * h + 2]) + v.z);
            r[4 * h + 3] = __float_as_uint(__uint_as_float(r[4 * h + 3]) + v.w);
          }
        emit(std::integral_constant<int, 1>(), r, o.row0 + 8 * g, scale0(o) + 8 * g, feature0(o), min(8, o.rows - 8 * g));
      }
    }
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }

  if (group >= 0 && gtid == 0) bulk_wait_group0();  // C is written before the CTA ends
  // A pair's MMAs read both CTAs' shared memory and write both TMEMs: neither
  // CTA leaves before both are done.
  tc_fence_before();
  if (kPair)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    if (kPair)
      tmem_dealloc_pair(tmem_base, kTmemCols);
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

size_t fixed_smem(int out_size, bool gate, int experts) {
  const int staged = kChunk * (gate ? 64 : 128) * out_size * staging_bufs(out_size);
  return 1024 /* alignment */ + kGroups * (staged + (gate ? 512 * 16 : 0)) + (3 * kMaxStages + 6) * 8 + 8 +
         3 * (static_cast<size_t>(experts) + 1) * 4;
}

template <typename OutT, bool kGate, Mode kMode>
cudaError_t launch(const MxGemmArgs& g, const Params& p, size_t smem, int grid, cudaStream_t stream, const char** why) {
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  auto kernel = mx_gemm_kernel<OutT, kGate, kMode>;
  if (dev >= 64 || !attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_done[dev] = true;
  }
  CUtensorMap tw, tw2, tx, txs, tc;
  const uint64_t k2 = g.K / 2, n = g.N;
  const uint32_t wbox = kGate ? 64 : 128;
  if (!make_tma_3d_u8(&tw, g.b, k2, n, g.experts, k2, k2 * n, kBKBytes, wbox) ||
      (kGate && !make_tma_3d_u8(&tw2, g.b2, k2, n, g.experts, k2, k2 * n, kBKBytes, wbox)) ||
      !make_tma_3d_u8(&tx, g.a, k2, g.rows, 1, k2, k2 * g.rows, kBKBytes, kMode == kPairs ? p.tn / 2 : p.tn) ||
      !make_tma_3d_u8(&txs, g.a, k2, g.rows, 1, k2, k2 * g.rows, kBKBytes, kSmallBox) ||
      (p.tma && !make_tma_3d_u8(&tc, g.c, n * sizeof(OutT), g.rows, 1, g.ldc * sizeof(OutT),
                                g.ldc * sizeof(OutT) * g.rows, 128, kChunk))) {
    *why = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  const int cluster = kMode == kSplitK ? p.splits : kMode == kPairs ? 2 : 1;
  return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, stream, cluster, tw, kGate ? tw2 : tw, tx, txs,
                    p.tma ? tc : tx, p);
}

template <typename OutT, bool kGate>
cudaError_t launch_mode(const MxGemmArgs& g, const Params& p, size_t smem, int grid, cudaStream_t stream,
                        const char** why) {
  return p.splits > 1 ? launch<OutT, kGate, kSplitK>(g, p, smem, grid, stream, why)
         : p.pair     ? launch<OutT, kGate, kPairs>(g, p, smem, grid, stream, why)
                      : launch<OutT, kGate, kWhole>(g, p, smem, grid, stream, why);
}

template <typename OutT>
cudaError_t launch_out(const MxGemmArgs& g, const Params& p, size_t smem, int grid, cudaStream_t stream,
                       const char** why) {
  return g.b2 ? launch_mode<OutT, true>(g, p, smem, grid, stream, why)
              : launch_mode<OutT, false>(g, p, smem, grid, stream, why);
}

// Tile shapes, and what a K tile and the rest of a tile take, in us, when every SM
// has one: fitted to 285 products of 1 .. 6000 tokens (up to 1024 per expert) with
// weights of 1024x16384 .. 14336x4096, each timed in every shape, so that the shape
// chosen is the fastest or close to it (0.5 % slower on the mean, 7 % at worst).  A
// tile of few tokens is bound by the loads of its weights; of the large ones a pair's
// need half the token bytes; 256 tokens have one accumulator, and their epilogue
// waits.  (Tiles of 160 and 224 tokens were never
// faster by more than 4 %.)
struct Shape {
  int tn, pair;
  double k_tile_us, tile_us;
};
constexpr Shape kShapes[] = {{32, 0, 0.17, 1.2}, {64, 0, 0.21, 0.9}, {128, 0, 0.23, 1.15},
                             {128, 1, 0.22, 1.4}, {192, 1, 0.27, 1.25}, {256, 1, 0.34, 2.4}};

// 128-row scale blocks that a tile of tn tokens can touch: an expert's tiles begin
// at multiples of tn, a multiple of 32, so at up to four places within a block.
constexpr int tile_scale_blocks(int tn) {
  int most = 0;
  for (int i = 0; i < 4; ++i) {
    const int blocks = ((i * tn % 128) + tn - 1) / 128 + 1;
    most = blocks > most ? blocks : most;
  }
  return most;
}
// TMEM columns of the token scales of 128 K columns.
constexpr int tile_scale_cols(int tn) { return tn <= 128 ? 4 : tn / 32; }
// What the kernel takes for granted of a shape: the scale writers hold the words of
// two scale blocks and store 4, 6 or 8 of them (224 tokens that begin at row 96 of a
// block touch three, and have 7).
constexpr bool shapes_fit() {
  for (const Shape& s : kShapes) {
    const int cols = tile_scale_cols(s.tn);
    if (s.tn % 32 || s.tn > 256 || tile_scale_blocks(s.tn) > 2 || (cols != 4 && cols != 6 && cols != 8)) return false;
  }
  return true;
}
static_assert(shapes_fit(), "a tile shape that the kernel is not made for");

// CTAs that share the K of each of at most `tiles` tiles.  A call of one tile per SM
// takes 4 + 0.17 us per K tile (launch, set-up and first loads are in the 4; kShapes
// has what a tile adds to a round); sharing K costs some 1.5 us more for the exchange
// and divides the rest until HBM is the limit (some 65 SMs).  Measured, one token:
// 1024x16384 14.1 -> 8.9 us with 4 CTAs and 8.0 with 8, 2048x7168 8.4 -> 7.0 with 4,
// 7168x16384 17.2 -> 15.9 with 2; but 4096x7168 8.6 with 1, 2 and 4, 7168x12288 13.0
// -> 13.1 with 2, 2048x2048 5.1 -> 5.7 with 4.  Clusters that find no room wait for
// others to end: 33 of 4 (4224x7168) took 8.8 us and 34 14.1, 9 of 8 8.3 and 16 15.6.
int k_splits(int64_t tiles, int KT, int num_sms) {
  return tiles * 8 <= num_sms / 2 && KT >= 48 ? 8
         : tiles * 5 <= num_sms && KT >= 24     ? 4
         : tiles * 2 <= num_sms && KT >= 56     ? 2
                                                : 1;
}

// Output features of a tile.
int tile_features(bool gate, int pair) { return (gate ? 64 : 128) * (pair ? 2 : 1); }

// Experts that can have a row.
int busy_experts(const MxGemmArgs& g) { return g.experts < g.rows ? g.experts : g.rows; }

// Tiles at most, whatever the offsets.
int64_t most_tiles(const MxGemmArgs& g, int tn, int busy, int n_tiles) {
  return g.offsets ? (static_cast<int64_t>(g.rows) / tn + busy) * n_tiles
                   : (static_cast<int64_t>(g.rows) + tn - 1) / tn * n_tiles;
}

// The shape with the shortest rounds of tiles.  How unevenly a routing fills the
// experts is not known here: tiles are counted for 0.6 .. 1.5 times the mean.
Shape choose_shape(const MxGemmArgs& g, bool gate, int KT, int busy, int num_sms) {
  const double mean = static_cast<double>(g.rows) / busy;
  Shape best = kShapes[0];
  double best_us = 1e30;
  for (const Shape& s : kShapes) {
    const int features = tile_features(gate, s.pair);
    double per_expert = 0;
    if (g.offsets)
      for (const double f : {0.6, 0.8, 1.0, 1.2, 1.5}) per_expert += std::ceil(f * mean / s.tn) / 5;
    else
      per_expert = std::ceil(mean / s.tn);
    const int n_tiles = (g.N + features - 1) / features;
    const int splits = s.pair ? 1 : k_splits(most_tiles(g, s.tn, busy, n_tiles), KT, num_sms);
    const double tiles = per_expert * busy * n_tiles;
    const double us = splits > 1 ? KT * s.k_tile_us / splits + s.tile_us + 1.5
                                 : std::ceil(tiles / (s.pair ? num_sms / 2 : num_sms)) * (KT * s.k_tile_us + s.tile_us);
    if (us < best_us) {
      best = s;
      best_us = us;
    }
  }
  return best;
}

}  // namespace

MxGemmShape mx_gemm_shape(const MxGemmArgs& g, int num_sms) {
  const bool gate = g.b2 != nullptr;
  const int KT = (g.K + kBK - 1) / kBK, busy = busy_experts(g);
  const Shape s = choose_shape(g, gate, KT, busy, num_sms);
  const int features = tile_features(gate, s.pair), n_tiles = (g.N + features - 1) / features;
  return MxGemmShape{s.tn, s.pair, s.pair ? 1 : k_splits(most_tiles(g, s.tn, busy, n_tiles), KT, num_sms)};
}

cudaError_t launch_mx_gemm(const MxGemmArgs& g, int num_sms, cudaStream_t stream, const char** why) {
  const bool gate = g.b2 != nullptr;
  const int out_size = g.out_dtype == 2 ? 4 : g.out_dtype == 3 ? 1 : 2;
  Params p{};
  p.sfw = static_cast<const uint8_t*>(g.sfb);
  p.sfw2 = static_cast<const uint8_t*>(g.sfb2);
  p.sfx = static_cast<const uint8_t*>(g.sfa);
  p.c = g.c;
  p.c_scales = static_cast<uint8_t*>(g.c_scales);
  p.offsets = g.offsets;
  p.rows = g.rows;
  p.N = g.N;
  p.K = g.K;
  p.experts = g.experts;
  p.ldc = g.ldc;
  p.status = g.status;
  p.inject = g.inject;
  p.vec = g.out_dtype != 3 && reinterpret_cast<uintptr_t>(g.c) % 16 == 0 && g.ldc * out_size % 16 == 0;
  // (A TMA store ends its rows at multiples of 16 bytes only, and its coordinates are
  // bytes here, in 32 bits.)
  const int64_t row_bytes = static_cast<int64_t>(g.N) * out_size;
  p.tma = p.vec && row_bytes % 16 == 0 && row_bytes < INT32_MAX - 1024;
  const MxGemmShape shape = mx_gemm_shape(g, num_sms);
  p.tn = shape.tn;
  p.pair = shape.pair;
  p.splits = shape.splits;
  const int features = tile_features(gate, shape.pair);
  p.n_tiles = (g.N + features - 1) / features;
  const int x_rows = p.pair ? p.tn / 2 : p.tn;  // token rows in a CTA's shared memory
  p.nblk = tile_scale_blocks(p.tn);
  p.acc_bufs = p.tn <= 192 ? 2 : 1;
  p.x_cols = tile_scale_cols(p.tn);
  p.sf_cols = 8 + 2 * p.x_cols;
  const int64_t exact = most_tiles(g, p.tn, busy_experts(g), p.n_tiles);
  // Stages: what shared memory and TMEM hold.
  const size_t fixed = fixed_smem(out_size, gate, g.experts) + (p.splits > 1 ? sums_bytes(p.tn, p.splits) : 0);
  const size_t stage = kABytes + x_rows * kBKBytes + ((gate ? 2 : 1) + p.nblk) * kSfBytes;
  int stages = static_cast<int>((kSmemMax - fixed) / stage);
  const int tmem_stages = (kTmemCols - p.acc_bufs * p.tn) / p.sf_cols;
  stages = stages < tmem_stages ? stages : tmem_stages;
  p.stages = stages < kMaxStages ? stages : kMaxStages;
  // A producer waits on a stage by phase parity, which is exact only while it
  // waits for every stage at most one lap behind: not more producers than stages.
  p.producers = p.stages < kMaxProducers ? p.stages : kMaxProducers;
  const int64_t workers = p.pair ? num_sms / 2 : num_sms;
  const int64_t grid = p.splits > 1 ? exact * p.splits : (exact < workers ? exact : workers) * (p.pair ? 2 : 1);
  const size_t smem = fixed + p.stages * stage;
  return g.out_dtype == 0   ? launch_out<__half>(g, p, smem, static_cast<int>(grid), stream, why)
         : g.out_dtype == 1 ? launch_out<__nv_bfloat16>(g, p, smem, static_cast<int>(grid), stream, why)
         : g.out_dtype == 3 ? launch_mode<Codes, true>(g, p, smem, static_cast<int>(grid), stream, why)
                            : launch_out<float>(g, p, smem, static_cast<int>(grid), stream, why);
}

}  // namespace nvfp4
