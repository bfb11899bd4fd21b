// Weights to the 4-bit format of fp4.h and back.  No reference counterpart.
//
// Both touch each value once and are bound by memory: a 16-bit value costs 2.53 bytes, a 32-bit one 4.53.  50,304 x 1,024 from bf16
// (130 MB) 21.5 us, 6.1 TB/s, and back 19.9; 8,192 x 1,024 from fp32 (38 MB) 6.2 us and 9.5.
#include <algorithm>

#include "fp4.h"

namespace atma {

struct Fp4QuantArgs {
  const void* w;  // (N, K), row stride ldw (written when dequantizing)
  int64_t ldw;
  uint8_t* data;  // (N, K / 2), row stride ldd
  int64_t ldd;
  uint8_t* scale;  // (N, K / 32), row stride lds
  int64_t lds;
  int64_t N;
  int K;
  int parts;  // 512-column parts of a row
};

// the largest of the four lanes of a quad
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));
}

// A wave takes 512 columns of a row, 8 consecutive values a lane: a group is the four lanes of a quad, its maximum two lane
// exchanges on the magnitudes' bits (as integers infinities and NaN lie above every number)
template <typename T>
__global__ void __launch_bounds__(256) quantize_fp4_kernel(Fp4QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t n = item / a.parts;
  if (n >= a.N) return;
  const int c = (int)(item - n * a.parts) * 512 + lane * 8;
  float v[8] = {};
  if (c < a.K) {
    const T* p = (const T*)a.w + n * a.ldw + c;
    if constexpr (sizeof(T) == 4) {
      const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
    } else {
      const u32x4 u = *(const u32x4*)p;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = elem16<T>(u, e);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
  const int code = fp4_scale_code(quad_max(top));
  if (c >= a.K) return;
  const float s = fp4_scale(code);
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], s, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], s, 3);
  *(uint32_t*)(a.data + n * a.ldd + c / 2) = o;
  if ((lane & 3) == 0) a.scale[n * a.lds + c / kFp4Group] = (uint8_t)code;
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_fp4_kernel(Fp4QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t n = item / a.parts;
  if (n >= a.N) return;
  const int c = (int)(item - n * a.parts) * 512 + lane * 8;
  if (c >= a.K) return;
  const uint32_t w = *(const uint32_t*)(a.data + n * a.ldd + c / 2);
  const float s = fp4_scale(a.scale[n * a.lds + c / kFp4Group]);
  T* p = (T*)a.w + n * a.ldw + c;
  if constexpr (sizeof(T) == 4) {
    const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    *(f32x4*)p = f32x4{v0[0], v0[1], v1[0], v1[1]};
    *(f32x4*)(p + 4) = f32x4{v2[0], v2[1], v3[0], v3[1]};
  } else {
    *(u32x4*)p = fp4_unpack8<T>(w, s);
  }
}

static int weight_fp4(const char* what, bool back, const void* w, int64_t ldw, const void* data, int64_t ldd, const void* scale,
                      int64_t lds, int64_t N, int64_t K, int dtype, void* stream) {
  const int size = dtype_size(dtype);
  if (!size) return set_error(ATMA_ERR_UNSUPPORTED, "%s: fp32 or 16-bit weights (dtype %d)", what, dtype);
  if (N < 0 || K < kFp4Group || K % kFp4Group || K > (1 << 24) || N > 0x7fffffff)
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: K must be a multiple of 32 up to 2^24, N below 2^31 (N=%lld K=%lld)", what,
                     (long long)N, (long long)K);
  if (N == 0) return ATMA_OK;
  if (!w || !data || !scale) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)w % 16 || (ldw * size) % 16 || ldw < K || (uintptr_t)data % 4 || ldd % 4 || ldd < K / 2 || lds < K / kFp4Group)
    return set_error(ATMA_ERR_INVALID, "%s: rows of the weights must be 16-byte aligned, rows of data 4-byte", what);
  Fp4QuantArgs a{w, ldw, (uint8_t*)data, ldd, (uint8_t*)scale, lds, N, (int)K, (int)((K + 511) / 512)};
  // a wave for each 512 columns of a row; a launch holds fewer than 2^32 threads, so what no one launch holds goes in several
  const int64_t rows = ((1 << 24) - 1) * 4ll / a.parts;
  for (int64_t n = 0; n < N; n += rows) {
    Fp4QuantArgs p = a;
    p.N = std::min(rows, N - n);
    p.w = (const char*)w + n * ldw * size;
    p.data += n * ldd;
    p.scale += n * lds;
    const dim3 grid((unsigned)((p.N * a.parts + 3) / 4));
    auto launch = [&](auto zero) {
      using T = decltype(zero);
      if (back) dequantize_fp4_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(p);
      else quantize_fp4_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    };
    if (dtype == ATMA_BF16) launch(bf16{});
    else if (dtype == ATMA_F16) launch(f16{});
    else launch(float{});
  }
  return check_launch(what);
}

}  // namespace atma

extern "C" int atma_quantize_weight_fp4(const void* w, int64_t ldw, void* data, int64_t ldd, void* scale, int64_t lds, int64_t N,
                                        int64_t K, int dtype, void* stream) {
  return atma::weight_fp4("quantize_weight_fp4", false, w, ldw, data, ldd, scale, lds, N, K, dtype, stream);
}

extern "C" int atma_dequantize_weight_fp4(const void* data, int64_t ldd, const void* scale, int64_t lds, void* w, int64_t ldw,
                                          int64_t N, int64_t K, int dtype, void* stream) {
  return atma::weight_fp4("dequantize_weight_fp4", true, w, ldw, data, ldd, scale, lds, N, K, dtype, stream);
}
