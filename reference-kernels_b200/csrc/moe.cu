// Tokens sorted by expert and back.
//
// Every token has `top` slots, each with an expert's number.  sort gives each
// slot that has one of the experts 0 .. E-1 a row, by expert and, within an
// expert, in the order of the slots; other numbers (negative, or an expert of
// another rank) are not routed.
//   gather            xs[row] = x[token]
//   gather_backward   dx[token] = sum over its rows of dxs[row]
//   combine           y[token] = sum over its slots of w[slot] * ys[row]
//   combine_backward  dys[row] = w[slot] * dy[token],  dw[slot] = <dy[token], ys[row]>
// Sums are held in fp32, in the order of the slots, and rounded once; no
// value is added with atomics, so results do not change from run to run.
// Rows outside offsets[0] .. offsets[E] - 1 belong to nobody, whatever the slots
// say: they are not read, and written as zeros.
//
// All of them are bound by memory.  The work is split by token and not by row:
// a token's own row is then read (gather, combine_backward) or written
// (combine, gather_backward) once, not `top` times, and no two threads write
// the same place.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kernels.h"

namespace nvfp4 {
namespace {

// ------------------------------------------------------------------ sort
// A stable counting sort.  A CTA takes a run of slots and each of its 32 warps
// a part of that run; within a warp 32 slots at a time are ranked by ballots.
// hist[warp][expert] in shared memory first counts, then (after sums over the warps,
// the CTAs and the experts) holds the next free row.
// One CTA does short lists, a cluster of eight longer ones, whose CTAs read one
// another's counts from distributed shared memory.  Lists that keep a cluster's
// warps busy for long take a second launch, before it, that counts each CTA's run
// to memory (counts[cta][expert]), and a CTA per SM at most.
constexpr int kSortWarps = 32;
constexpr int kSortThreads = 32 * kSortWarps;

constexpr int kSortCluster = 8;

__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename Id>
__device__ __forceinline__ int expert_id(const Id* ids, int slot, int E) {
  const Id v = ids[slot];
  return v >= 0 && v < E ? static_cast<int>(v) : -1;
}

// The lanes that hold the same id (-1 .. E - 1): one ballot per bit.  (A
// match.any took about 1 us for a step of 32 warps.)
__device__ __forceinline__ uint32_t same_id(int id, int E) {
  uint32_t peers = 0xffffffffu;
  for (int bit = 1; bit <= E; bit <<= 1) {  // -1 counts as E
    const bool set = (id < 0 ? E : id) & bit;
    const uint32_t with = __ballot_sync(0xffffffffu, set);
    peers &= set ? with : ~with;
  }
  return peers;
}

// Calls f(slot, id) for this warp's part of the run [begin, end), 32 slots at a
// time (id -1: not routed, or behind the end), with the loads of four such steps
// in flight together.
template <typename Id, typename F>
__device__ __forceinline__ void for_run(const Id* ids, int begin, int end, int E, F f) {
  constexpr int kAhead = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = ((end - begin + kSortThreads - 1) / kSortThreads) * 32;  // slots per warp
  const int b = begin + warp * per, e = min(b + per, end);
  for (int s0 = b; s0 < e; s0 += 32 * kAhead) {
    int id[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int slot = s0 + 32 * k + lane;
      id[k] = slot < e ? expert_id(ids, slot, E) : -1;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (s0 + 32 * k < e) f(s0 + 32 * k + lane, id[k], e);
  }
}

// Counts the run [begin, end) into hist[warp][E].
template <typename Id>
__device__ __forceinline__ void count_run(const Id* ids, int begin, int end, int E, int* hist) {
  int* mine = hist + (threadIdx.x >> 5) * E;
  for_run(ids, begin, end, E, [&](int, int id, int) {
    if (id >= 0) atomicAdd(mine + id, 1);  // counts alone: their order does not matter
  });
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) moe_count_kernel(const MoeSortArgs a) {
  extern __shared__ int hist[];
  if (threadIdx.x == 0) pdl_allow_dependents();
  for (int i = threadIdx.x; i < kSortWarps * a.experts; i += kSortThreads) hist[i] = 0;
  pdl_wait();
  __syncthreads();
  const int begin = blockIdx.x * a.run, end = min(begin + a.run, a.slots_n);
  count_run(static_cast<const Id*>(a.ids), begin, end, a.experts, hist);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kSortThreads) {
    int n = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) n += hist[w * a.experts + e];
    a.counts[blockIdx.x * a.experts + e] = n;
  }
}

template <typename Id, bool kCluster>
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const MoeSortArgs a) {
  extern __shared__ int hist[];
  __shared__ int cta_count[kCluster ? kMaxExperts : 1];
  __shared__ int warp_sum[kSortWarps];
  __shared__ int routed;
  if (threadIdx.x == 0) pdl_allow_dependents();
  const int E = a.experts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * E; i += kSortThreads) hist[i] = 0;
  pdl_wait();
  __syncthreads();
  const int begin = blockIdx.x * a.run, end = min(begin + a.run, a.slots_n);
  const Id* ids = static_cast<const Id*>(a.ids);
  count_run(ids, begin, end, E, hist);
  __syncthreads();
  // Thread e: expert e's total, and its slots in the CTAs before this one.
  const int e = threadIdx.x;
  int total = 0, before = 0;
  if (kCluster) {
    int mine = 0;
    if (e < E) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) mine += hist[w * E + e];
      cta_count[e] = mine;
    }
    cluster_sync_all();
    if (e < E) {
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        const int n = ld_cluster(map_peer(smem_u32(&cta_count[e]), c));
        total += n;
        before += c < static_cast<int>(blockIdx.x) ? n : 0;
      }
    }
  } else if (e < E) {
    if (gridDim.x == 1) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) total += hist[w * E + e];
    } else {
#pragma unroll 8
      for (int c = 0; c < static_cast<int>(gridDim.x); ++c) {
        const int n = a.counts[c * E + e];
        total += n;
        before += c < static_cast<int>(blockIdx.x) ? n : 0;
      }
    }
  }
  // Exclusive sum of the totals over the experts (E <= the CTA's threads).
  int sum = total;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += o;
    }
    warp_sum[lane] = s;
  }
  __syncthreads();
  const int first = sum - total + (warp ? warp_sum[warp - 1] : 0);
  if (e < E) {
    if (blockIdx.x == 0) {
      a.offsets[e] = first;
      if (e == E - 1) a.offsets[E] = first + total;
    }
    if (e == E - 1) routed = first + total;
    int next = first + before;
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = hist[w * E + e];
      hist[w * E + e] = next;
      next += n;
    }
  }
  __syncthreads();
  int* mine = hist + warp * E;
  for_run(ids, begin, end, E, [&](int slot, int id, int stop) {
    const uint32_t peers = same_id(id, E);
    const int rank = __popc(peers & ((1u << lane) - 1));
    int row = -1;
    if (id >= 0) row = mine[id] + rank;
    __syncwarp();
    if (id >= 0 && rank == 0) mine[id] += __popc(peers);
    __syncwarp();
    if (slot < stop) a.slots[slot] = row;
    if (row >= 0) a.order[row] = slot;
  });
  if (kCluster) cluster_sync_all();  // the others have read this CTA's counts
  // Rows that no slot has.
  for (int i = routed + blockIdx.x * kSortThreads + threadIdx.x; i < a.slots_n; i += gridDim.x * kSortThreads)
    a.order[i] = -1;
}

// ------------------------------------------------------------------ rows
// N elements that are loaded and stored together: 16 bytes where rows and bases
// allow it, else as many as divide the row and its address.  Held as whole
// words: as an array of 16-bit values the compiler gave each a register.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = sizeof(T) * N;
  using Word = std::conditional_t<kBytes == 2, uint16_t, uint32_t>;
  struct alignas(kBytes) Raw {
    Word w[kBytes / sizeof(Word)];
  } raw;

  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(raw.w[i]);
    } else {
      const uint32_t half = kBytes == 2 ? raw.w[0] : (i & 1 ? raw.w[i / 2] >> 16 : raw.w[i / 2] & 0xffffu);
      if constexpr (std::is_same<T, __half>::value)
        return __half2float(__ushort_as_half(static_cast<unsigned short>(half)));
      else
        return __uint_as_float(half << 16);
    }
  }
  // All N at once, from fp32.
  __device__ __forceinline__ void set(const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) raw.w[i] = __float_as_uint(v[i]);
    } else if constexpr (N == 1) {
      raw.w[0] = bits(v[0]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) raw.w[i] = bits(v[2 * i]) | bits(v[2 * i + 1]) << 16;
    }
  }

 private:
  static __device__ __forceinline__ uint32_t bits(float v) {
    if constexpr (std::is_same<T, __half>::value)
      return __half_as_ushort(__float2half_rn(v));
    else
      return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
};

constexpr int kRowThreads = 128;
// Packs per thread and step: `bytes` of loads in flight.
template <typename T, int N>
__host__ __device__ constexpr int in_flight(int bytes) {
  return bytes / static_cast<int>(sizeof(T) * N) < 16 ? bytes / static_cast<int>(sizeof(T) * N) : 16;
}

// The rows [lo, hi) that the experts have, within the `rows` that there are
// (without offsets, which the sums over a token's rows may lack: all).
struct Range {
  int lo, hi;
  __device__ __forceinline__ bool has(int row) const { return row >= lo && row < hi; }
};
__device__ __forceinline__ Range experts_rows(const MoeRowArgs& a) {
  const int rows = a.tokens * a.top;
  if (!a.offsets) return Range{0, rows};
  const int lo = min(max(a.offsets[0], 0), rows);
  return Range{lo, min(max(a.offsets[a.experts], lo), rows)};
}

// Zeroes the rows of out [rows][H] that no expert has, in front of the range and
// behind it.  The slots write rows of the range alone, so that no row is written
// by two CTAs.
template <typename T, int N>
__device__ __forceinline__ void zero_others(T* out, Range of, int rows, int packs) {
  const int64_t front = static_cast<int64_t>(of.lo) * packs, own = static_cast<int64_t>(of.hi - of.lo) * packs;
  const int64_t n = static_cast<int64_t>(rows) * packs - own;
  Pack<T, N> z;
  const float zeros[N] = {};
  z.set(zeros);
  Pack<T, N>* const dst = reinterpret_cast<Pack<T, N>*>(out);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    dst[i < front ? i : i + own] = z;
}

// A unit is one token and kRowThreads * kU packs of its row.
template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads) moe_gather_kernel(const MoeRowArgs a) {
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  constexpr int kU = in_flight<T, N>(16);
  const int packs = a.hidden / N;
  const int per_row = (packs + kRowThreads * kU - 1) / (kRowThreads * kU);
  const int64_t units = static_cast<int64_t>(a.tokens) * per_row;
  const Range of = experts_rows(a);
  T* const out = static_cast<T*>(a.out);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int t = static_cast<int>(u / per_row);
    const int p0 = static_cast<int>(u - static_cast<int64_t>(t) * per_row) * kRowThreads * kU + threadIdx.x;
    const Pack<T, N>* src =
        reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) + static_cast<int64_t>(t) * a.in_stride);
    Pack<T, N> v[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i)
      if (p0 + i * kRowThreads < packs) v[i] = src[p0 + i * kRowThreads];
    for (int j = 0; j < a.top; ++j) {
      const int row = a.slots[static_cast<int64_t>(t) * a.top + j];
      if (!of.has(row)) continue;
      Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(out) + static_cast<int64_t>(row) * packs;
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (p0 + i * kRowThreads < packs) dst[p0 + i * kRowThreads] = v[i];
    }
  }
  zero_others<T, N>(out, of, a.tokens * a.top, packs);
}

// combine (kWeighted) and gather_backward: a token's rows, weighted or not, added
// up.  Four rows at a time: their places and weights first, then the loads of all
// four together, then the sums in the order of the slots.
template <typename T, int N, bool kWeighted>
__global__ void __launch_bounds__(kRowThreads) moe_reduce_kernel(const MoeRowArgs a) {
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  constexpr int kU = in_flight<T, N>(N * sizeof(T) == 16 ? 32 : 16), kJ = 4;
  const int packs = a.hidden / N;
  const int per_row = (packs + kRowThreads * kU - 1) / (kRowThreads * kU);
  const int64_t units = static_cast<int64_t>(a.tokens) * per_row;
  const Range of = experts_rows(a);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int t = static_cast<int>(u / per_row);
    const int p0 = static_cast<int>(u - static_cast<int64_t>(t) * per_row) * kRowThreads * kU + threadIdx.x;
    float acc[kU][N];
#pragma unroll
    for (int i = 0; i < kU; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) acc[i][n] = 0.f;
    for (int j0 = 0; j0 < a.top; j0 += kJ) {
      int row[kJ];
      float w[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int64_t slot = static_cast<int64_t>(t) * a.top + j0 + j;
        row[j] = j0 + j < a.top ? a.slots[slot] : -1;
        w[j] = kWeighted && j0 + j < a.top ? a.weights[slot] : 1.f;
      }
      Pack<T, N> v[kJ][kU];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const Pack<T, N>* src = reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) +
                                                                    static_cast<int64_t>(row[j]) * a.in_stride);
#pragma unroll
        for (int i = 0; i < kU; ++i)
          if (of.has(row[j]) && p0 + i * kRowThreads < packs) v[j][i] = src[p0 + i * kRowThreads];
      }
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (of.has(row[j]))
#pragma unroll
          for (int i = 0; i < kU; ++i)
#pragma unroll
            for (int n = 0; n < N; ++n)
              acc[i][n] = kWeighted ? fmaf(w[j], v[j][i].get(n), acc[i][n]) : acc[i][n] + v[j][i].get(n);
    }
    Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(static_cast<T*>(a.out)) + static_cast<int64_t>(t) * packs;
#pragma unroll
    for (int i = 0; i < kU; ++i)
      if (p0 + i * kRowThreads < packs) {
        Pack<T, N> v;
        v.set(acc[i]);
        dst[p0 + i * kRowThreads] = v;
      }
  }
}

// kLanes threads take one slot: dys = w * dy and the product <dy, ys>, summed
// over them in a fixed order.  A warp per slot where there are many (dy comes
// from L1 for a token's other slots), a CTA per slot where there are few: 16
// tokens of 8 slots and 7168 took 16.2 us with a CTA per token.
template <typename T, int N, int kLanes>
__global__ void __launch_bounds__(kRowThreads) moe_combine_backward_kernel(const MoeRowArgs a) {
  static_assert(kLanes == 32 || kLanes == kRowThreads, "a warp or the CTA");
  __shared__ float part[kRowThreads / 32];
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  constexpr int kU = in_flight<T, N>(64);
  const int packs = a.hidden / N;
  const int rows = a.tokens * a.top;
  const Range of = experts_rows(a);
  const int lane = threadIdx.x % kLanes;
  T* const out = static_cast<T*>(a.out);
  constexpr int kSlots = kRowThreads / kLanes;  // per CTA and step
  for (int64_t slot = static_cast<int64_t>(blockIdx.x) * kSlots + threadIdx.x / kLanes; slot < rows;
       slot += static_cast<int64_t>(gridDim.x) * kSlots) {
    const int row = a.slots[slot];
    if (!of.has(row)) {  // the same for all kLanes threads
      if (lane == 0) a.dweights[slot] = 0.f;
      continue;
    }
    const int64_t t = slot / a.top;
    const float w = a.weights[slot];
    const Pack<T, N>* dy =
        reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.grad) + t * a.grad_stride);
    const Pack<T, N>* ys =
        reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) + static_cast<int64_t>(row) * a.in_stride);
    Pack<T, N>* dys = reinterpret_cast<Pack<T, N>*>(out) + static_cast<int64_t>(row) * packs;
    float dot = 0.f;
    for (int p0 = lane; p0 < packs; p0 += kLanes * kU) {
      Pack<T, N> g[kU], v[kU];
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (p0 + i * kLanes < packs) {
          g[i] = dy[p0 + i * kLanes];
          v[i] = ys[p0 + i * kLanes];
        }
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (p0 + i * kLanes < packs) {
          float scaled[N];
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const float gf = g[i].get(n);
            dot = fmaf(gf, v[i].get(n), dot);
            scaled[n] = w * gf;
          }
          Pack<T, N> d;
          d.set(scaled);
          dys[p0 + i * kLanes] = d;
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (kLanes == 32) {
      if (lane == 0) a.dweights[slot] = dot;
    } else {
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kRowThreads / 32; ++i) s += part[i];
        a.dweights[slot] = s;
      }
      __syncthreads();
    }
  }
  zero_others<T, N>(out, of, rows, packs);
}

template <typename T, int N>
cudaError_t launch_rows(MoeRowOp op, const MoeRowArgs& a, int num_sms, cudaStream_t stream) {
  const int packs = a.hidden / N;
  const int step = kRowThreads * in_flight<T, N>(op != kMoeGather && N * sizeof(T) == 16 ? 32 : 16);
  const int64_t slots = static_cast<int64_t>(a.tokens) * a.top;
  const bool warps = op == kMoeCombineBackward && slots >= 8 * num_sms;  // enough for a warp each to fill the SMs
  const int64_t units = op == kMoeCombineBackward ? (warps ? (slots + 3) / 4 : slots)
                                                  : static_cast<int64_t>(a.tokens) * ((packs + step - 1) / step);
  // (64 CTAs of 128 threads per SM against 16, 8192 tokens to 4 experts each, bf16,
  // 4096: gather 62 -> 55 us, combine 55 -> 52, its gradient 97 -> 93.)
  const int64_t cap = static_cast<int64_t>(num_sms) * 64;
  const dim3 grid(static_cast<unsigned>(units < cap ? units : cap)), block(kRowThreads);
  switch (op) {
    case kMoeGather:
      return launch_pdl(moe_gather_kernel<T, N>, grid, block, 0, stream, 1, a);
    case kMoeGatherBackward:
      return launch_pdl(moe_reduce_kernel<T, N, false>, grid, block, 0, stream, 1, a);
    case kMoeCombine:
      return launch_pdl(moe_reduce_kernel<T, N, true>, grid, block, 0, stream, 1, a);
    default:
      return warps ? launch_pdl(moe_combine_backward_kernel<T, N, 32>, grid, block, 0, stream, 1, a)
                   : launch_pdl(moe_combine_backward_kernel<T, N, kRowThreads>, grid, block, 0, stream, 1, a);
  }
}

// The widest pack that divides the rows and every address.
template <typename T>
cudaError_t launch_type(MoeRowOp op, const MoeRowArgs& a, int num_sms, cudaStream_t stream) {
  uintptr_t all = static_cast<uintptr_t>(a.hidden) * sizeof(T) | static_cast<uintptr_t>(a.in_stride) * sizeof(T) |
                  reinterpret_cast<uintptr_t>(a.in) | reinterpret_cast<uintptr_t>(a.out);
  if (op == kMoeCombineBackward)
    all |= static_cast<uintptr_t>(a.grad_stride) * sizeof(T) | reinterpret_cast<uintptr_t>(a.grad);
  if (all % 16 == 0) return launch_rows<T, 16 / sizeof(T)>(op, a, num_sms, stream);
  if (sizeof(T) == 2 && all % 4 == 0) return launch_rows<T, 4 / sizeof(T)>(op, a, num_sms, stream);
  return launch_rows<T, 1>(op, a, num_sms, stream);
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t smem) {
  if (smem <= 40 * 1024) return cudaSuccess;  // (with the static part under the default 48 KB)
  constexpr int kMost = kSortWarps * kMaxExperts * static_cast<int>(sizeof(int));
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
}

template <typename Id>
cudaError_t launch_sort(const MoeSortArgs& a, int ctas, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kSortWarps) * a.experts * sizeof(int);
  cudaError_t e;
  if (ctas == kSortCluster) {
    if ((e = allow_smem(moe_sort_kernel<Id, true>, smem)) != cudaSuccess) return e;
    return launch_pdl(moe_sort_kernel<Id, true>, dim3(ctas), dim3(kSortThreads), smem, stream, kSortCluster, a);
  }
  if ((e = allow_smem(moe_sort_kernel<Id, false>, smem)) != cudaSuccess) return e;
  if (ctas > 1) {
    if ((e = allow_smem(moe_count_kernel<Id>, smem)) != cudaSuccess) return e;
    e = launch_pdl(moe_count_kernel<Id>, dim3(ctas), dim3(kSortThreads), smem, stream, 1, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(moe_sort_kernel<Id, false>, dim3(ctas), dim3(kSortThreads), smem, stream, 1, a);
}

// CTAs for n slots, by measured times (us): 512 slots 3.3 in one CTA and 4.1 in a
// cluster, 2048 4.4 and 3.8; 32768 7.0 in a cluster and 6.5 in 32 CTAs with a second
// launch, 131072 18.2 and 9.1; 524288 20.4 in 32 CTAs and 13.2 in 148.
int sort_ctas(int n, int num_sms) {
  if (n <= 1024) return 1;
  if (n <= 32768) return kSortCluster;
  const int c = n / 4096 < 32 ? 32 : n / 4096;
  return c < num_sms ? c : num_sms;
}

}  // namespace

size_t moe_sort_workspace_bytes(int n, int experts, int num_sms) {
  const int c = sort_ctas(n, num_sms);
  return c > kSortCluster ? static_cast<size_t>(c) * experts * sizeof(int) : 0;
}

cudaError_t launch_moe_sort(MoeSortArgs a, int num_sms, cudaStream_t stream) {
  const int ctas = sort_ctas(a.slots_n, num_sms);
  a.run = (a.slots_n + ctas - 1) / ctas;
  return a.id_bytes == 8 ? launch_sort<int64_t>(a, ctas, stream) : launch_sort<int32_t>(a, ctas, stream);
}

cudaError_t launch_moe_rows(MoeRowOp op, const MoeRowArgs& a, int num_sms, cudaStream_t stream) {
  return a.dtype == 0   ? launch_type<__half>(op, a, num_sms, stream)
         : a.dtype == 1 ? launch_type<__nv_bfloat16>(op, a, num_sms, stream)
                        : launch_type<float>(op, a, num_sms, stream);
}

}  // namespace nvfp4
