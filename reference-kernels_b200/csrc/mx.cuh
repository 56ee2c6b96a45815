// Conversions between fp32 and MXFP4 (mx_quant.cu has the rule).
#pragma once

#include <stdint.h>

namespace nvfp4 {

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

// Two: lo in the low nibble.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
  uint16_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u16.u8 %0, t;\n\t}"
      : "=h"(r)
      : "f"(hi), "f"(lo));
  return r;
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

}  // namespace nvfp4
