// The 4-bit weight format of the quantizer and products: bytes of two float4 e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives; the even k in the low half), each group of 32 along a row with a power-of-two scale (float8_e8m0fnu code
// c, scale 2^(c - 127); code 255: every value of the group is NaN).
//
// The scale of a group is the smallest 2^e, e in [-125, 125], that brings its largest magnitude to 7 or less: the values
// between 6 and 7 round to 6, the nearest there is.  Signal to noise on normally distributed values is 19.03 dB, against 18.75
// where nothing may pass 6, 18.78 for e = floor(log2(largest)) - 2, and 19.05 for the better of two neighbouring scales in
// each group.  The instructions that convert two such values to 16 bits (v_cvt_scalef32_pk_{bf16,f16}_fp4) multiply by a power of two on the
// way, so a product's operands are the weights themselves and no sum is ever rescaled.
#pragma once

#include "common.h"

namespace atma {

constexpr int kFp4Group = 32;

// code = 127 + e for the bits of a largest magnitude m 2^E, m in [1, 2): e = E - 2 where m <= 1.75, else E - 1
__device__ __forceinline__ int fp4_scale_code(uint32_t top) {
  if (top >= 0x7f800000u) return 255;  // an infinity or NaN in the group
  return min(max((int)((top + 0x1fffffu) >> 23) - 2, 2), 252);
}
__device__ __forceinline__ float fp4_scale(int code) { return __builtin_bit_cast(float, (uint32_t)code << 23); }

// Eight values (low half of the low byte first) times 2^e as 16-bit values, exact wherever T holds them
template <typename T>
__device__ __forceinline__ u32x4 fp4_unpack8(uint32_t w, float scale) {
  if constexpr (__is_same(T, bf16)) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  } else {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
  }
}

}  // namespace atma
