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
// Sums are held in fp32, in the order of the slots, and rounded once; nothing
// is added with atomics, so results do not change from run to run.
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
// a part of that run; within a warp 32 slots at a time are ranked with
// match_any.  hist[warp][expert] in shared memory first counts, then (after
// sums over the warps, the CTAs and the experts) holds the next free row.
// One CTA does short lists in one launch; longer ones take a second launch,
// before it, that counts each CTA's run (counts[cta][expert]), and each CTA
// adds up the counts of the CTAs before it itself.
constexpr int kSortWarps = 32;
constexpr int kSortThreads = 32 * kSortWarps;

template <typename Id>
__device__ __forceinline__ int expert_id(const Id* ids, int slot, int E) {
  const Id v = ids[slot];
  return v >= 0 && v < E ? static_cast<int>(v) : -1;
}

// Counts the run [begin, end) into hist[warp][E].
template <typename Id>
__device__ __forceinline__ void count_run(const Id* ids, int begin, int end, int E, int* hist) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* mine = hist + warp * E;
  const int per = ((end - begin + kSortThreads - 1) / kSortThreads) * 32;  // slots per warp
  const int b = begin + warp * per, e = min(b + per, end);
  for (int s0 = b; s0 < e; s0 += 32) {
    const int slot = s0 + lane;
    const int id = slot < e ? expert_id(ids, slot, E) : -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && (peers & ((1u << lane) - 1)) == 0) mine[id] += __popc(peers);
    __syncwarp();
  }
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

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const MoeSortArgs a) {
  extern __shared__ int hist[];
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
  if (e < E) {
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
  const int per = ((end - begin + kSortThreads - 1) / kSortThreads) * 32;
  const int b = begin + warp * per, stop = min(b + per, end);
  for (int s0 = b; s0 < stop; s0 += 32) {
    const int slot = s0 + lane;
    const int id = slot < stop ? expert_id(ids, slot, E) : -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(peers & ((1u << lane) - 1));
    int row = -1;
    if (id >= 0) row = mine[id] + rank;
    __syncwarp();
    if (id >= 0 && rank == 0) mine[id] += __popc(peers);
    __syncwarp();
    if (slot < stop) a.slots[slot] = row;
    if (row >= 0) a.order[row] = slot;
  }
  // Rows that no slot has.
  for (int i = routed + blockIdx.x * kSortThreads + threadIdx.x; i < a.slots_n; i += gridDim.x * kSortThreads)
    a.order[i] = -1;
}

// ------------------------------------------------------------------ rows
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(float& d, float v) { d = v; }

// N elements that are loaded and stored together: 16 bytes where rows and
// bases allow it, else as many as divide the row and its address.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

constexpr int kRowThreads = 128;
constexpr int kUnroll = 4;  // packs per thread and step: loads in flight

// Zeroes the rows of out [rows][H] that no slot has (from offsets[E] on).
template <typename T, int N>
__device__ __forceinline__ void zero_tail(T* out, const int* offsets, int E, int rows, int packs) {
  const int first = min(max(offsets[E], 0), rows);
  const int64_t n = static_cast<int64_t>(rows - first) * packs;
  Pack<T, N> z;
#pragma unroll
  for (int i = 0; i < N; ++i) put(z.v[i], 0.f);
  Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(out) + static_cast<int64_t>(first) * packs;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    dst[i] = z;
}

// A unit is one token and kRowThreads * kUnroll packs of its row.
template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads) moe_gather_kernel(const MoeRowArgs a) {
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int packs = a.hidden / N;
  const int per_row = (packs + kRowThreads * kUnroll - 1) / (kRowThreads * kUnroll);
  const int64_t units = static_cast<int64_t>(a.tokens) * per_row;
  const int rows = a.tokens * a.top;
  T* const out = static_cast<T*>(a.out);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int t = static_cast<int>(u / per_row);
    const int p0 = static_cast<int>(u - static_cast<int64_t>(t) * per_row) * kRowThreads * kUnroll + threadIdx.x;
    const Pack<T, N>* src =
        reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) + static_cast<int64_t>(t) * a.in_stride);
    Pack<T, N> v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (p0 + i * kRowThreads < packs) v[i] = src[p0 + i * kRowThreads];
    for (int j = 0; j < a.top; ++j) {
      const int row = a.slots[static_cast<int64_t>(t) * a.top + j];
      if (row < 0 || row >= rows) continue;
      Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(out) + static_cast<int64_t>(row) * packs;
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (p0 + i * kRowThreads < packs) dst[p0 + i * kRowThreads] = v[i];
    }
  }
  zero_tail<T, N>(out, a.offsets, a.experts, rows, packs);
}

// combine (kWeighted) and gather_backward: a token's rows, weighted or not, added up.
template <typename T, int N, bool kWeighted>
__global__ void __launch_bounds__(kRowThreads) moe_reduce_kernel(const MoeRowArgs a) {
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  constexpr int kU = 2;
  const int packs = a.hidden / N;
  const int per_row = (packs + kRowThreads * kU - 1) / (kRowThreads * kU);
  const int64_t units = static_cast<int64_t>(a.tokens) * per_row;
  const int rows = a.tokens * a.top;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int t = static_cast<int>(u / per_row);
    const int p0 = static_cast<int>(u - static_cast<int64_t>(t) * per_row) * kRowThreads * kU + threadIdx.x;
    float acc[kU][N];
#pragma unroll
    for (int i = 0; i < kU; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) acc[i][n] = 0.f;
#pragma unroll 4
    for (int j = 0; j < a.top; ++j) {
      const int64_t slot = static_cast<int64_t>(t) * a.top + j;
      const int row = a.slots[slot];
      if (row < 0 || row >= rows) continue;
      const float w = kWeighted ? a.weights[slot] : 1.f;
      const Pack<T, N>* src =
          reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) + static_cast<int64_t>(row) * a.in_stride);
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (p0 + i * kRowThreads < packs) {
          const Pack<T, N> v = src[p0 + i * kRowThreads];
#pragma unroll
          for (int n = 0; n < N; ++n) acc[i][n] = kWeighted ? fmaf(w, to_float(v.v[n]), acc[i][n]) : acc[i][n] + to_float(v.v[n]);
        }
    }
    Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(static_cast<T*>(a.out)) + static_cast<int64_t>(t) * packs;
#pragma unroll
    for (int i = 0; i < kU; ++i)
      if (p0 + i * kRowThreads < packs) {
        Pack<T, N> v;
#pragma unroll
        for (int n = 0; n < N; ++n) put(v.v[n], acc[i][n]);
        dst[p0 + i * kRowThreads] = v;
      }
  }
}

// A CTA takes one token: for each of its slots, dys = w * dy and the product
// <dy, ys>, summed over the threads in a fixed order.
template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads) moe_combine_backward_kernel(const MoeRowArgs a) {
  __shared__ float part[kRowThreads / 32];
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int packs = a.hidden / N;
  const int rows = a.tokens * a.top;
  T* const out = static_cast<T*>(a.out);
  for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const Pack<T, N>* dy =
        reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.grad) + static_cast<int64_t>(t) * a.grad_stride);
    for (int j = 0; j < a.top; ++j) {
      const int64_t slot = static_cast<int64_t>(t) * a.top + j;
      const int row = a.slots[slot];
      if (row < 0 || row >= rows) {  // the same for the whole CTA
        if (threadIdx.x == 0) a.dweights[slot] = 0.f;
        continue;
      }
      const float w = a.weights[slot];
      const Pack<T, N>* ys =
          reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(a.in) + static_cast<int64_t>(row) * a.in_stride);
      Pack<T, N>* dys = reinterpret_cast<Pack<T, N>*>(out) + static_cast<int64_t>(row) * packs;
      float dot = 0.f;
#pragma unroll kUnroll
      for (int p = threadIdx.x; p < packs; p += kRowThreads) {
        const Pack<T, N> g = dy[p], v = ys[p];
        Pack<T, N> d;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float gf = to_float(g.v[n]);
          dot = fmaf(gf, to_float(v.v[n]), dot);
          put(d.v[n], w * gf);
        }
        dys[p] = d;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
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
  zero_tail<T, N>(out, a.offsets, a.experts, rows, packs);
}

template <typename T, int N>
cudaError_t launch_rows(MoeRowOp op, const MoeRowArgs& a, int num_sms, cudaStream_t stream) {
  const int packs = a.hidden / N;
  const int step = kRowThreads * (op == kMoeGather ? kUnroll : 2);
  const int64_t units =
      op == kMoeCombineBackward ? a.tokens : static_cast<int64_t>(a.tokens) * ((packs + step - 1) / step);
  const int64_t cap = static_cast<int64_t>(num_sms) * 16;
  const dim3 grid(static_cast<unsigned>(units < cap ? units : cap)), block(kRowThreads);
  switch (op) {
    case kMoeGather:
      return launch_pdl(moe_gather_kernel<T, N>, grid, block, 0, stream, 1, a);
    case kMoeGatherBackward:
      return launch_pdl(moe_reduce_kernel<T, N, false>, grid, block, 0, stream, 1, a);
    case kMoeCombine:
      return launch_pdl(moe_reduce_kernel<T, N, true>, grid, block, 0, stream, 1, a);
    default:
      return launch_pdl(moe_combine_backward_kernel<T, N>, grid, block, 0, stream, 1, a);
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

template <typename Id>
cudaError_t launch_sort(const MoeSortArgs& a, int ctas, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(kSortWarps) * a.experts * sizeof(int);
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(moe_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSortWarps * kMaxExperts * sizeof(int));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(moe_count_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kSortWarps * kMaxExperts * sizeof(int));
    if (e != cudaSuccess) return e;
  }
  if (ctas > 1) {
    cudaError_t e = launch_pdl(moe_count_kernel<Id>, dim3(ctas), dim3(kSortThreads), smem, stream, 1, a);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(moe_sort_kernel<Id>, dim3(ctas), dim3(kSortThreads), smem, stream, 1, a);
}

// CTAs for n slots: one up to 4096 (four passes of its 1024 threads: a second
// launch and the counts' trip through memory cost more), then 2048 slots each,
// at most one CTA per SM.
int sort_ctas(int n, int num_sms) {
  if (n <= 4096) return 1;
  const int c = (n + 2047) / 2048;
  return c < num_sms ? c : num_sms;
}

}  // namespace

size_t moe_sort_workspace_bytes(int n, int experts, int num_sms) {
  const int c = sort_ctas(n, num_sms);
  return c > 1 ? static_cast<size_t>(c) * experts * sizeof(int) : 0;
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
