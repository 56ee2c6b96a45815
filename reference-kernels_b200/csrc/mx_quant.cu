// MXFP4 quantiser and its reverse: e2m1 values with one power-of-two scale
// (e8m0: 2^(code - 127), 255 = NaN) per 32 elements, as the OCP microscaling
// format defines it.
//
//   e   = floor(log2(max |x|)) - 2, at least -127          (2 = exponent of e2m1's largest binade)
//   q_i = e2m1_rn_satfinite(x_i * 2^-e),  code = e + 127
// A power of two divides exactly, so each q_i is the correctly rounded quotient
// (ties to even, above 6 saturates to 6).  A zero block gets code 0; a NaN or
// an infinity in a block gets code 255 and zero codes: the whole block reads as
// NaN.  Scales are written 128x4-blocked (mx_scale_word), columns past K / 32
// of the last word as 0.
//
// All kernels here are bound by HBM: 2 (4) bytes read and 17/32 byte written per
// 16-bit (32-bit) element, the reverse for dequantize.  Along the rows a lane
// takes one block: 64 (128) bytes in 32-byte loads, all in flight at once, 16
// bytes of codes; the scale codes of four lanes meet in one 4-byte store.  Rows
// are padded to four blocks in the numbering of the lanes, so that those four
// always lie in one row.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kernels.h"
#include "mx.cuh"

namespace nvfp4 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}

__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The 32 elements of a block as they lie in memory.
template <typename T>
struct Block {
  static constexpr int kWords = 8 * sizeof(T);
  alignas(16) uint32_t w[kWords];  // (loaded in 16-byte pieces)

  // kAlign: bytes that the address is a multiple of, 32 or 16.
  template <int kAlign>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kAlign == 32) {
#pragma unroll
      for (int i = 0; i < kWords / 8; ++i) load32(reinterpret_cast<const uint32_t*>(p) + 8 * i, w + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        *reinterpret_cast<uint4*>(w + 4 * i) = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
  }
  // Any address: the warp loads its lanes' blocks one after another, an element
  // per lane and all in flight, and deals them out through `rows` of shared memory.
  // (4096 x 4096 in bf16: 15.8 us, 35 with each lane loading its own elements; 6.5
  // for aligned rows.)
  static constexpr int kPitch = 32 + 4 / static_cast<int>(sizeof(T));  // elements; an odd number of words
  __device__ __forceinline__ void load_any(const T* p, bool active, T (*rows)[kPitch]) {
    const int lane = threadIdx.x & 31;
    const uint32_t with = __ballot_sync(0xffffffffu, active);
    __syncwarp();  // the last step's rows are read
    T v[32];
#pragma unroll
    for (int b = 0; b < 32; ++b) {
      const T* q = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), b));
      v[b] = with >> b & 1 ? q[lane] : T(0.f);
    }
#pragma unroll
    for (int b = 0; b < 32; ++b) rows[b][lane] = v[b];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint32_t*>(rows[lane])[i];
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (std::is_same<T, float>::value) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i >> 1] >> (16 * (i & 1)))));
    } else {
      return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
  }
  // Bits of the largest magnitude, as fp32: magnitudes are ordered like their
  // bits, NaN above infinity.
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = max(m >> 16, m & 0xffffu);
      return std::is_same<T, __half>::value
                 ? __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))))
                 : m << 16;
    }
  }
  // The block's codes at scale 2^(code - 127).
  __device__ __forceinline__ uint4 codes(uint32_t code) const;
};

template <typename T>
__device__ __forceinline__ uint4 Block<T>::codes(uint32_t code) const {
  if (code == 255u) return make_uint4(0, 0, 0, 0);
  const float inv = inverse_scale(code);
  uint32_t q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (*this)[8 * k + i] * inv;
    q[k] = e2m1x8(v);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

struct Rows {
  int row[kMaxExperts + 1], blk[kMaxExperts + 1];
};

// The scale row of row r of rows sorted by expert; -1 where no expert has it.
__device__ __forceinline__ int64_t sorted_scale_row(const Rows& tab, int experts, int r) {
  const int e = expert_of(tab.row, experts, r);
  return e == experts || r < tab.row[0] ? -1 : static_cast<int64_t>(tab.blk[e]) * 128 + (r - tab.row[e]);
}

// kMode: 0 rows (rows_per of each of `experts` matrices), 1 rows sorted by
// expert, 2 tokens written to each of their sorted rows.
template <typename T, int kMode, int kAlign>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const MxQuantArgs a) {
  __shared__ Rows tab;
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  if (kMode != 0) {
    if (threadIdx.x < 32) load_expert_table(a.offsets, a.experts, a.sorted_rows, tab.row, tab.blk);
    __syncthreads();
  }
  const int K32 = a.K >> 5, K128 = (a.K + 127) >> 7;
  const uint32_t total = static_cast<uint32_t>(a.rows) * (4 * K128);
  uint8_t* const packed = static_cast<uint8_t*>(a.packed);
  uint8_t* const scales = static_cast<uint8_t*>(a.scales);
  for (uint32_t f0 = blockIdx.x * kThreads + threadIdx.x - lane; f0 < total; f0 += gridDim.x * kThreads) {
    const uint32_t f = f0 + lane;
    const int r = static_cast<int>(f / (4 * K128)), j = static_cast<int>(f - r * (4 * K128));
    bool active = f < total && j < K32;
    int64_t src = static_cast<int64_t>(r) * a.x_rstride, scale_row = r;
    if (kMode == 0 && a.rows_per != a.rows) {
      const int e = r / a.rows_per, i = r - e * a.rows_per;
      src = e * a.x_estride + static_cast<int64_t>(i) * a.x_rstride;
      scale_row = static_cast<int64_t>(e) * ((a.rows_per + 127) >> 7) * 128 + i;
    }
    Block<T> x;
    const T* const p = static_cast<const T*>(a.x) + src + 32 * j;
    if constexpr (kAlign == 1) {
      __shared__ alignas(16) T rows[kWarps][32][Block<T>::kPitch];
      x.load_any(p, active, rows[threadIdx.x >> 5]);
    } else {
      if (active) x.template load<kAlign>(p);
    }
    if (kMode == 1) {
      scale_row = f < total ? sorted_scale_row(tab, a.experts, r) : -1;
      active = active && scale_row >= 0;
    }
    const uint32_t code = active ? scale_code(x.amax_bits()) : 0u;
    uint4 q = make_uint4(0, 0, 0, 0);
    if (active) q = x.codes(code);
    uint32_t word = code << (8 * (lane & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    if (kMode != 2) {
      if (active) {
        *reinterpret_cast<uint4*>(packed + static_cast<int64_t>(r) * (a.K >> 1) + 16 * j) = q;
        if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(scale_row, j >> 2, K128)) = word;
      }
    } else {
      // A warp within one token: lane t finds the scale row of the token's t-th
      // slot for all.  Else every lane for itself.
      const bool one = __all_sync(0xffffffffu, r == __shfl_sync(0xffffffffu, r, 0)) && f0 + 31 < total;
      for (int t0 = 0; t0 < a.top; t0 += 32) {
        const int nt = min(32, a.top - t0);
        int row = -1;
        int64_t srow = -1;
        if (one && lane < nt) {
          row = a.slots[static_cast<int64_t>(r) * a.top + t0 + lane];
          srow = row < 0 ? -1 : sorted_scale_row(tab, a.experts, row);
        }
        for (int t = 0; t < nt; ++t) {
          int out;
          int64_t s;
          if (one) {
            out = __shfl_sync(0xffffffffu, row, t);
            s = __shfl_sync(0xffffffffu, srow, t);
          } else {
            out = active ? a.slots[static_cast<int64_t>(r) * a.top + t0 + t] : -1;
            s = out < 0 ? -1 : sorted_scale_row(tab, a.experts, out);
          }
          if (s < 0 || !active) continue;
          *reinterpret_cast<uint4*>(packed + static_cast<int64_t>(out) * (a.K >> 1) + 16 * j) = q;
          if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(s, j >> 2, K128)) = word;
        }
      }
    }
  }
}

// Blocks down the columns of x [rows][cols]; the result is the quantised
// transpose [cols][rows padded to 32], rows past the end as zeros.  A CTA takes
// 256 rows x 64 columns: warp w the 32 rows of block w, a lane two neighbouring
// columns of them (kVec: one load per row, 128 bytes per warp for 16-bit types),
// the loads of 32 rows in flight together.  (With the row check around each load
// they went one by one: 143 us for 8192 x 7168 in bf16, against 23 of traffic.)
// The codes pass through shared memory so that 128 contiguous bytes are written
// per column: 16-byte pieces straight from the registers would fill half a
// sector each.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) mx_quantize_columns_kernel(const MxQuantArgs a) {
  __shared__ uint4 codes[64][kWarps + 1];
  struct alignas(4) Scales {  // of a column, stored to memory as words
    uint8_t code[kWarps];
  };
  __shared__ Scales sc[64];
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = a.rows, C = a.K;  // a.K holds the number of columns here
  const int Kt = (R + 31) & ~31;  // K of the result
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 256 + warp * 32;
  const int c = c0 + 2 * lane;
  struct alignas(2 * sizeof(T)) Two {
    T v[2];
  };
  Two v[32];
  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(r0) * a.x_rstride + c;
  if (kVec && r0 + 32 <= R && c < C) {  // (kVec: C is even)
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = *reinterpret_cast<const Two*>(x + i * a.x_rstride);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[i].v[h] = T(0.f);
        if (r0 + i < R && c + h < C) v[i].v[h] = x[i * a.x_rstride + h];
      }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // This column's block, put together as it would lie along a row.
    Block<T> b;
#pragma unroll
    for (int i = 0; i < 32; ++i) reinterpret_cast<T*>(b.w)[i] = v[i].v[h];
    const uint32_t code = scale_code(b.amax_bits());
    codes[2 * lane + h][warp] = b.codes(code);
    sc[2 * lane + h].code[warp] = r0 < Kt ? static_cast<uint8_t>(code) : 0;
  }
  __syncthreads();
  const int k0 = blockIdx.y * 256;
  uint8_t* const packed = static_cast<uint8_t*>(a.packed);
#pragma unroll
  for (int i = threadIdx.x; i < 64 * kWarps; i += kThreads) {
    const int col = i / kWarps, w = i % kWarps;
    if (c0 + col < C && k0 + w * 32 < Kt)
      *reinterpret_cast<uint4*>(packed + static_cast<int64_t>(c0 + col) * (Kt >> 1) + ((k0 + w * 32) >> 1)) =
          codes[col][w];
  }
  const int K128 = (Kt + 127) >> 7;
  if (threadIdx.x < 128) {
    const int col = threadIdx.x >> 1, j = threadIdx.x & 1;
    if (c0 + col < C && (k0 >> 7) + j < K128)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.scales) + mx_scale_word(c0 + col, (k0 >> 7) + j, K128)) =
          reinterpret_cast<const uint32_t*>(sc[col].code)[j];
  }
}

// Codes and scales back to values, a block per lane.  kMode as above (0, 1);
// rows that no expert has are written as zeros.
template <typename T, int kMode>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const MxQuantArgs a) {
  __shared__ Rows tab;
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  if (kMode != 0) {
    if (threadIdx.x < 32) load_expert_table(a.offsets, a.experts, a.sorted_rows, tab.row, tab.blk);
    __syncthreads();
  }
  const int K32 = a.K >> 5, K128 = (a.K + 127) >> 7;
  const uint32_t total = static_cast<uint32_t>(a.rows) * K32;
  for (uint32_t f = blockIdx.x * kThreads + threadIdx.x; f < total; f += gridDim.x * kThreads) {
    const int r = static_cast<int>(f / K32), j = static_cast<int>(f - r * K32);
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.packed) + 16 * static_cast<int64_t>(f));
    int64_t scale_row = r;
    if (kMode == 0 && a.rows_per != a.rows) {
      const int e = r / a.rows_per, i = r - e * a.rows_per;
      scale_row = static_cast<int64_t>(e) * ((a.rows_per + 127) >> 7) * 128 + i;
    }
    if (kMode == 1) scale_row = sorted_scale_row(tab, a.experts, r);
    const bool here = kMode == 0 || scale_row >= 0;
    const float s =
        here ? scale_value(static_cast<const uint8_t*>(a.scales)[mx_scale_word(scale_row, j >> 2, K128) + (j & 3)]) : 0.f;
    Block<T> out;
    T* const o = reinterpret_cast<T*>(out.w);
    const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t h[4];
      e2m1x8_to_f16x2x4(words[k], h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        o[8 * k + 2 * i] = from_float<T>(here ? v.x * s : 0.f);
        o[8 * k + 2 * i + 1] = from_float<T>(here ? v.y * s : 0.f);
      }
    }
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(const_cast<void*>(a.x)) + 32 * static_cast<int64_t>(f));
#pragma unroll
    for (int i = 0; i < Block<T>::kWords / 8; ++i) store32(dst + 8 * i, out.w + 8 * i);
  }
}

template <typename T, int kMode>
cudaError_t quantize_mode(const MxQuantArgs& a, int align, dim3 grid, cudaStream_t stream) {
  const dim3 block(kThreads);
  return align == 32   ? launch_pdl(mx_quantize_kernel<T, kMode, 32>, grid, block, 0, stream, 1, a)
         : align == 16 ? launch_pdl(mx_quantize_kernel<T, kMode, 16>, grid, block, 0, stream, 1, a)
                       : launch_pdl(mx_quantize_kernel<T, kMode, 1>, grid, block, 0, stream, 1, a);
}

template <typename T>
cudaError_t quantize_rows(const MxQuantArgs& a, int align, dim3 grid, cudaStream_t stream) {
  return a.slots     ? quantize_mode<T, 2>(a, align, grid, stream)
         : a.offsets ? quantize_mode<T, 1>(a, align, grid, stream)
                     : quantize_mode<T, 0>(a, align, grid, stream);
}

template <typename T>
cudaError_t quantize_columns(const MxQuantArgs& a, bool vec, cudaStream_t stream) {
  const dim3 grid((a.K + 63) / 64, (a.rows + 255) / 256), block(kThreads);
  if (vec) return launch_pdl(mx_quantize_columns_kernel<T, true>, grid, block, 0, stream, 1, a);
  return launch_pdl(mx_quantize_columns_kernel<T, false>, grid, block, 0, stream, 1, a);
}

template <typename T>
cudaError_t dequantize_rows(const MxQuantArgs& a, dim3 grid, cudaStream_t stream) {
  const dim3 block(kThreads);
  if (a.offsets) return launch_pdl(mx_dequantize_kernel<T, 1>, grid, block, 0, stream, 1, a);
  return launch_pdl(mx_dequantize_kernel<T, 0>, grid, block, 0, stream, 1, a);
}

// A CTA of 256 threads per 256 blocks, up to per_sm of them per SM; the rest in
// strides.  Rows want many (64 against 16 per SM: 8192x7168 24.6 -> 23.8 us,
// dequantized 26.2 -> 23.9), tokens of sorted rows few, since every CTA builds the
// table of the experts (4 against 16: 8192 tokens to 4 experts each 31.4 -> 29.1).
dim3 row_grid(const MxQuantArgs& a, int num_sms, int per_sm) {
  const int64_t lanes = static_cast<int64_t>(a.rows) * ((a.K + 127) / 128 * 4);
  const int64_t blocks = (lanes + kThreads - 1) / kThreads, cap = static_cast<int64_t>(num_sms) * per_sm;
  return dim3(static_cast<unsigned>(blocks < cap ? blocks : cap));
}

}  // namespace

cudaError_t launch_mx_quantize(const MxQuantArgs& a, int num_sms, cudaStream_t stream) {
  const int size = a.dtype == 2 ? 4 : 2;
  const uintptr_t base = reinterpret_cast<uintptr_t>(a.x);
  if (a.columns) {
    const bool vec = a.K % 2 == 0 && a.x_rstride % 2 == 0 && base % (2 * size) == 0;
    return a.dtype == 0   ? quantize_columns<__half>(a, vec, stream)
           : a.dtype == 1 ? quantize_columns<__nv_bfloat16>(a, vec, stream)
                          : quantize_columns<float>(a, vec, stream);
  }
  const uint64_t all = base | static_cast<uint64_t>(a.x_rstride * size) | static_cast<uint64_t>(a.x_estride * size);
  const int align = all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : 1;
  const dim3 grid = row_grid(a, num_sms, a.slots ? 4 : a.offsets ? 16 : 64);
  return a.dtype == 0   ? quantize_rows<__half>(a, align, grid, stream)
         : a.dtype == 1 ? quantize_rows<__nv_bfloat16>(a, align, grid, stream)
                        : quantize_rows<float>(a, align, grid, stream);
}

cudaError_t launch_mx_dequantize(const MxQuantArgs& a, int num_sms, cudaStream_t stream) {
  const dim3 grid = row_grid(a, num_sms, 64);
  return a.dtype == 0   ? dequantize_rows<__half>(a, grid, stream)
         : a.dtype == 1 ? dequantize_rows<__nv_bfloat16>(a, grid, stream)
                        : dequantize_rows<float>(a, grid, stream);
}

}  // namespace nvfp4
