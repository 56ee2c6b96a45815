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
// takes 16 elements (one or two 16-byte loads in flight per array, 8 bytes of
// codes), two lanes a block, a warp 512 elements; the four scale codes of 128
// elements meet in one 4-byte store.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "kernels.h"

namespace nvfp4 {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 512;  // elements of a row per warp step

// Eight floats -> eight e2m1 codes, element 0 in the low nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
      "mov.b32 %0, {t0, t1, t2, t3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }

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

// N consecutive elements as floats; kVec: 16-byte loads (aligned).
template <int N, bool kVec, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
  if constexpr (kVec) {
    constexpr int kPer = 16 / sizeof(T);
    uint4 w[N / kPer];
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_float(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_float(p[i]);
  }
}

// Largest magnitude as bits: ordered like the magnitudes, NaN above infinity.
template <int N>
__device__ __forceinline__ uint32_t amax_bits(const float (&v)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// Scale code of a block: the exponent field of the largest magnitude, less 2.
__device__ __forceinline__ uint32_t scale_code(uint32_t amax) {
  const uint32_t f = amax >> 23;
  return f == 255u ? 255u : f > 2u ? f - 2u : 0u;
}
// What the block's values are multiplied with: 2^(127 - code); 0 for a NaN block.
__device__ __forceinline__ float inverse_scale(uint32_t code) {
  return code == 255u ? 0.f : __uint_as_float((254u - code) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7fffffffu) : code == 0u ? __uint_as_float(0x00400000u)
                                                                   : __uint_as_float(code << 23);
}

struct Rows {
  int row[kMaxExperts + 1], blk[kMaxExperts + 1];
};

// kMode: 0 rows (rows_per of each of `experts` matrices), 1 rows sorted by
// expert, 2 tokens written to each of their sorted rows.
template <typename T, int kMode, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) mx_quantize_kernel(const MxQuantArgs a) {
  __shared__ Rows tab;
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  if (kMode != 0) {
    if (threadIdx.x < 32) load_expert_table(a.offsets, a.experts, a.sorted_rows, tab.row, tab.blk);
    __syncthreads();
  }
  const int K128 = (a.K + 127) >> 7;
  const uint32_t per_row = (a.K + kUnit - 1) / kUnit;
  const uint32_t units = per_row * static_cast<uint32_t>(a.rows);
  uint8_t* const packed = static_cast<uint8_t*>(a.packed);
  uint8_t* const scales = static_cast<uint8_t*>(a.scales);
  for (uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < units; u += gridDim.x * kWarps) {
    const int r = static_cast<int>(u / per_row);
    const int k = static_cast<int>(u - r * per_row) * kUnit + lane * 16;
    int64_t src = static_cast<int64_t>(r) * a.x_rstride, scale_row = r;
    if (kMode == 0 && a.rows_per != a.rows) {
      const int e = r / a.rows_per, i = r - e * a.rows_per;
      src = e * a.x_estride + static_cast<int64_t>(i) * a.x_rstride;
      scale_row = static_cast<int64_t>(e) * ((a.rows_per + 127) >> 7) * 128 + i;
    }
    if (kMode == 1) {
      const int e = expert_of(tab.row, a.experts, r);
      if (e == a.experts || r < tab.row[0]) continue;
      scale_row = static_cast<int64_t>(tab.blk[e]) * 128 + (r - tab.row[e]);
    }
    float v[16];
    if (k < a.K) {
      load_n<16, kVec>(static_cast<const T*>(a.x) + src + k, v);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    uint32_t m = amax_bits(v);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t code = scale_code(m);
    const float inv = inverse_scale(code);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = code == 255u ? 0.f : v[i] * inv;
    const uint2 q = make_uint2(e2m1x8(v), e2m1x8(v + 8));
    uint32_t word = code << (8 * ((lane >> 1) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    const int j = k >> 7;
    const bool has_word = (lane & 7) == 0 && k < a.K;
    if (kMode != 2) {
      if (k < a.K) *reinterpret_cast<uint2*>(packed + static_cast<int64_t>(r) * (a.K >> 1) + (k >> 1)) = q;
      if (has_word) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(scale_row, j, K128)) = word;
    } else {
      // Lane t finds the scale row of the token's t-th slot; all lanes then
      // write the codes to each.
      for (int t0 = 0; t0 < a.top; t0 += 32) {
        const int nt = min(32, a.top - t0);
        int row = -1;
        int64_t srow = 0;
        if (lane < nt) row = a.slots[static_cast<int64_t>(r) * a.top + t0 + lane];
        if (row >= 0) {
          const int e = expert_of(tab.row, a.experts, row);
          if (e == a.experts || row < tab.row[0])
            row = -1;
          else
            srow = static_cast<int64_t>(tab.blk[e]) * 128 + (row - tab.row[e]);
        }
        for (int t = 0; t < nt; ++t) {
          const int out = __shfl_sync(0xffffffffu, row, t);
          const int64_t s = __shfl_sync(0xffffffffu, srow, t);
          if (out < 0) continue;
          if (k < a.K) *reinterpret_cast<uint2*>(packed + static_cast<int64_t>(out) * (a.K >> 1) + (k >> 1)) = q;
          if (has_word) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(s, j, K128)) = word;
        }
      }
    }
  }
}

// Blocks down the columns of x [rows][cols]; the result is the quantised
// transpose [cols][rows padded to 32], rows past the end as zeros.  A CTA takes
// 256 rows x 64 columns: warp w the 32 rows of block w, a lane two neighbouring
// columns of them (kVec: one load per row, 128 bytes per warp for 16-bit
// types), 32 rows in registers.  The codes pass through shared memory so that
// 128 contiguous bytes are written per column: 16-byte pieces straight from the
// registers would fill half a sector each.
template <typename T, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) mx_quantize_columns_kernel(const MxQuantArgs a) {
  __shared__ uint4 codes[64][kWarps + 1];
  __shared__ uint8_t sc[64][kWarps];
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = a.rows, C = a.K;  // a.K holds the number of columns here
  const int Kt = (R + 31) & ~31;  // K of the result
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 256 + warp * 32;
  const int c = c0 + 2 * lane;
  float v[2][32];
  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(r0) * a.x_rstride + c;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[0][i] = v[1][i] = 0.f;
    if (r0 + i < R) {
      const T* p = x + static_cast<int64_t>(i) * a.x_rstride;
      if (kVec) {
        if (c < C) {  // C is even
          struct alignas(2 * sizeof(T)) Two {
            T v[2];
          };
          const Two t = *reinterpret_cast<const Two*>(p);
          v[0][i] = to_float(t.v[0]);
          v[1][i] = to_float(t.v[1]);
        }
      } else {
        if (c < C) v[0][i] = to_float(p[0]);
        if (c + 1 < C) v[1][i] = to_float(p[1]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t code = scale_code(amax_bits(v[h]));
    const float inv = inverse_scale(code);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[h][i] = code == 255u ? 0.f : v[h][i] * inv;
    codes[2 * lane + h][warp] = make_uint4(e2m1x8(v[h]), e2m1x8(v[h] + 8), e2m1x8(v[h] + 16), e2m1x8(v[h] + 24));
    sc[2 * lane + h][warp] = r0 < Kt ? static_cast<uint8_t>(code) : 0;
  }
  __syncthreads();
  const int k0 = blockIdx.y * 256;
  uint8_t* const packed = static_cast<uint8_t*>(a.packed);
  for (int i = threadIdx.x; i < 64 * kWarps; i += 32 * kWarps) {
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
          reinterpret_cast<const uint32_t*>(sc[col])[j];
  }
}

// Codes and scales back to values.  kMode as above (0, 1); rows behind the
// last expert's are written as zeros.
template <typename T, int kMode, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) mx_dequantize_kernel(const MxQuantArgs a) {
  __shared__ Rows tab;
  if (threadIdx.x == 0) pdl_allow_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  if (kMode != 0) {
    if (threadIdx.x < 32) load_expert_table(a.offsets, a.experts, a.sorted_rows, tab.row, tab.blk);
    __syncthreads();
  }
  const int K128 = (a.K + 127) >> 7;
  const uint32_t per_row = (a.K + kUnit - 1) / kUnit;
  const uint32_t units = per_row * static_cast<uint32_t>(a.rows);
  for (uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < units; u += gridDim.x * kWarps) {
    const int r = static_cast<int>(u / per_row);
    const int k = static_cast<int>(u - r * per_row) * kUnit + lane * 16;
    if (k >= a.K) continue;
    int64_t scale_row = r;
    bool here = true;
    if (kMode == 0 && a.rows_per != a.rows) {
      const int e = r / a.rows_per, i = r - e * a.rows_per;
      scale_row = static_cast<int64_t>(e) * ((a.rows_per + 127) >> 7) * 128 + i;
    }
    if (kMode == 1) {
      const int e = expert_of(tab.row, a.experts, r);
      here = e < a.experts && r >= tab.row[0];
      if (here) scale_row = static_cast<int64_t>(tab.blk[e]) * 128 + (r - tab.row[e]);
    }
    T out[16];
    if (here) {
      const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.packed) +
                                                      static_cast<int64_t>(r) * (a.K >> 1) + (k >> 1));
      const uint32_t word = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.scales) +
                                                               mx_scale_word(scale_row, k >> 7, K128));
      const float s = scale_value((word >> (8 * ((k >> 5) & 3))) & 255u);
      uint32_t h[8];
      e2m1x8_to_f16x2x4(q.x, *reinterpret_cast<uint32_t(*)[4]>(h));
      e2m1x8_to_f16x2x4(q.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        out[2 * i] = from_float<T>(f.x * s);
        out[2 * i + 1] = from_float<T>(f.y * s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) out[i] = from_float<T>(0.f);
    }
    T* dst = static_cast<T*>(const_cast<void*>(a.x)) + static_cast<int64_t>(r) * a.K + k;
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(out)[i];
  }
}

template <typename T>
cudaError_t quantize_rows(const MxQuantArgs& a, bool vec, dim3 grid, cudaStream_t stream) {
  const dim3 block(32 * kWarps);
  const int mode = a.slots ? 2 : a.offsets ? 1 : 0;
#define NVFP4_MX_QUANT(MODE, VEC) \
  if (mode == MODE && vec == VEC) return launch_pdl(mx_quantize_kernel<T, MODE, VEC>, grid, block, 0, stream, 1, a)
  NVFP4_MX_QUANT(0, true);
  NVFP4_MX_QUANT(0, false);
  NVFP4_MX_QUANT(1, true);
  NVFP4_MX_QUANT(1, false);
  NVFP4_MX_QUANT(2, true);
  NVFP4_MX_QUANT(2, false);
#undef NVFP4_MX_QUANT
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t quantize_columns(const MxQuantArgs& a, bool vec, cudaStream_t stream) {
  const dim3 grid((a.K + 63) / 64, (a.rows + 255) / 256), block(32 * kWarps);
  if (vec) return launch_pdl(mx_quantize_columns_kernel<T, true>, grid, block, 0, stream, 1, a);
  return launch_pdl(mx_quantize_columns_kernel<T, false>, grid, block, 0, stream, 1, a);
}

template <typename T>
cudaError_t dequantize_rows(const MxQuantArgs& a, dim3 grid, cudaStream_t stream) {
  const dim3 block(32 * kWarps);
  if (a.offsets) return launch_pdl(mx_dequantize_kernel<T, 1, true>, grid, block, 0, stream, 1, a);
  return launch_pdl(mx_dequantize_kernel<T, 0, true>, grid, block, 0, stream, 1, a);
}

dim3 row_grid(const MxQuantArgs& a, int num_sms) {
  const int64_t units = static_cast<int64_t>(a.rows) * ((a.K + kUnit - 1) / kUnit);
  const int64_t blocks = (units + kWarps - 1) / kWarps, cap = static_cast<int64_t>(num_sms) * 8;
  return dim3(static_cast<unsigned>(blocks < cap ? blocks : cap));
}

}  // namespace

cudaError_t launch_mx_quantize(const MxQuantArgs& a, int num_sms, cudaStream_t stream) {
  const int size = a.dtype == 2 ? 4 : 2;
  const auto bytes = [&](int64_t elements) { return elements * size; };
  const uintptr_t base = reinterpret_cast<uintptr_t>(a.x);
  if (a.columns) {
    const bool vec = a.K % 2 == 0 && a.x_rstride % 2 == 0 && base % (2 * size) == 0;
    return a.dtype == 0   ? quantize_columns<__half>(a, vec, stream)
           : a.dtype == 1 ? quantize_columns<__nv_bfloat16>(a, vec, stream)
                          : quantize_columns<float>(a, vec, stream);
  }
  const bool vec = base % 16 == 0 && bytes(a.x_rstride) % 16 == 0 && bytes(a.x_estride) % 16 == 0;
  const dim3 grid = row_grid(a, num_sms);
  return a.dtype == 0   ? quantize_rows<__half>(a, vec, grid, stream)
         : a.dtype == 1 ? quantize_rows<__nv_bfloat16>(a, vec, grid, stream)
                        : quantize_rows<float>(a, vec, grid, stream);
}

cudaError_t launch_mx_dequantize(const MxQuantArgs& a, int num_sms, cudaStream_t stream) {
  const dim3 grid = row_grid(a, num_sms);
  return a.dtype == 0   ? dequantize_rows<__half>(a, grid, stream)
         : a.dtype == 1 ? dequantize_rows<__nv_bfloat16>(a, grid, stream)
                        : dequantize_rows<float>(a, grid, stream);
}

}  // namespace nvfp4
