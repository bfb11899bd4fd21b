// The 8-bit format of the quantizers and products: float8_e4m3fn values, each block of 128 with a power-of-two scale
// (float8_e8m0fnu code c, scale 2^(c - 127)).
//
// The scale of a block is the smallest 2^e, e in [-126, 120], that brings its largest finite magnitude to 448 (1.75 * 2^8,
// the largest e4m3fn) or less.  A power of two keeps every product of values and scales exact, and the matrix
// instructions apply it themselves (v_mfma_scale), so no scale is ever multiplied in by vector instructions.  Values that
// are not finite do not enter a block's scale and are stored as NaN.
#pragma once

#include "common.h"

namespace atma {

constexpr int kFp8Block = 128;

// code = 127 + e for a largest magnitude m 2^E, m in [1, 2): e = E - 8 where m <= 1.75 (mantissa bits <= 0x600000), else
// E - 7; subnormal and zero magnitudes take the smallest scale
__device__ __forceinline__ int fp8_scale_code(float amax) {
  const int c = (int)((__builtin_bit_cast(uint32_t, amax) + 0x1fffffu) >> 23) - 8;
  return min(max(c, 1), 247);
}
// 2^(127 - code), a normal float for every code above
__device__ __forceinline__ float fp8_inv_scale(int code) {
  return __builtin_bit_cast(float, (uint32_t)(254 - code) << 23);
}
__device__ __forceinline__ float fp8_scale(int code) { return __builtin_bit_cast(float, (uint32_t)code << 23); }
// |x|, 0 where x is not finite
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;
}
// Four values to e4m3fn (round to nearest even; infinities and NaN to NaN), the first in the low byte
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return (uint32_t)v;
}
// Four values divided by a power of two to e4m3fn (v_cvt_scalef32_pk_fp8_f32), rounded as above
__device__ __forceinline__ uint32_t fp8_scaled4(float a, float b, float c, float d, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 v = {0, 0};
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, a, b, scale, false);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, v);
}

}  // namespace atma
