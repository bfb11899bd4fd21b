// Products with 4-bit weights: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]) for 16-bit x (M, K) and w (N, K) in the format of
// fp4.h, and the MLP's first projection with its activation, gate * relu(a)^2 of the fp32 sums.  No reference counterpart.
#include <algorithm>

#include "fp4.h"

namespace atma {

struct Fp4Args {
  const void* x;  // (M, K), row stride ldx
  int64_t ldx;
  const uint8_t* w;  // (N, K / 2) or, gated, (2 N, K / 2): the a rows, then the gate rows; row stride ldw
  int64_t ldw;
  const uint8_t* ws;  // the same rows, K / 32 codes each, row stride ldws
  int64_t ldws;
  const void* bias;  // (N,) or (2 N,), or null
  int bias_dtype;
  void* y;  // (M, N), row stride ldy
  int64_t ldy;
  int64_t M, N;
  int K;
};

__device__ __forceinline__ float fp4_bias(const Fp4Args& a, int64_t n) {
  if (!a.bias) return 0.f;
  if (a.bias_dtype == ATMA_F32) return ((const float*)a.bias)[n];
  if (a.bias_dtype == ATMA_BF16) return to_f32(((const bf16*)a.bias)[n]);
  return to_f32(((const f16*)a.bias)[n]);
}

// gate * relu(a)^2 in fp32 (v_maximum3_f32: NaN passes through, as torch's relu)
__device__ __forceinline__ float fp4_gate(float av, float gv) {
  const float pos = __builtin_elementwise_maximum(av, 0.f);
  return gv * (pos * pos);
}

// A wave owns 16 features x 16 tokens; lane (r, g) holds row r of both operands, k = 8 g .. + 7 of each 32
template <typename T, bool GATED>
__global__ void __launch_bounds__(64) fp4_kernel(Fp4Args a) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16;
  const T* x = (const T*)a.x + min(m0 + r, a.M - 1) * a.ldx + 8 * g;
  f32x4 acc[GATED ? 2 : 1] = {};
  for (int kb = 0; kb < a.K; kb += 32) {
    const u32x4 xv = *(const u32x4*)(x + kb);
#pragma unroll
    for (int t = 0; t < (GATED ? 2 : 1); ++t) {
      const int64_t n = min(f0 + r, a.N - 1) + t * a.N;
      const uint32_t w = *(const uint32_t*)(a.w + n * a.ldw + kb / 2 + 4 * g);
      acc[t] = mfma16x16x32<T>(fp4_unpack8<T>(w, fp4_scale(a.ws[n * a.ldws + kb / kFp4Group])), xv, acc[t]);
    }
  }
  const int64_t m = m0 + r;
  if (m >= a.M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t n = f0 + 4 * g + e;
    if (n >= a.N) break;
    float v = acc[0][e] + fp4_bias(a, n);
    if constexpr (GATED) v = fp4_gate(v, acc[1][e] + fp4_bias(a, a.N + n));
    ((T*)a.y)[m * a.ldy + n] = from_f32<T>(v);
  }
}

static int linear_fp4(const char* what, bool gated, Fp4Args a, int64_t K, int dtype, void* stream) {
  const int64_t rows = gated ? 2 * a.N : a.N;
  if (dtype != ATMA_BF16 && dtype != ATMA_F16)
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: 16-bit activations (dtype %d)", what, dtype);
  if (a.M < 0 || a.N < 1 || K < kFp4Group || K % kFp4Group || K > (1 << 22) || a.M > (1 << 30) || rows > (1 << 28))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: unsupported shape M=%lld N=%lld K=%lld (K a multiple of 32 up to 2^22, M up to "
                     "2^30, weight rows up to 2^28)", what, (long long)a.M, (long long)a.N, (long long)K);
  if (a.M == 0) return ATMA_OK;
  if (!a.x || !a.w || !a.ws || !a.y) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  a.K = (int)K;
  if (a.M == 1) a.ldx = K;  // (the stride of a single row means nothing)
  if (rows == 1) a.ldw = K / 2;
  if ((uintptr_t)a.x % 16 || a.ldx % 8 || a.ldx < K || (uintptr_t)a.w % 16 || a.ldw % 16 || a.ldw < K / 2)
    return set_error(ATMA_ERR_INVALID, "%s: rows of x and w must be 16-byte aligned and at least K long", what);
  if (a.ldws < 0) return set_error(ATMA_ERR_INVALID, "%s: negative stride of scales", what);
  // a tile's rows (at most 256) are addressed by 32-bit byte offsets
  if (a.ldx > (1 << 22) || a.ldw > (1 << 23))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: rows more than 8 MiB apart", what);
  if (a.bias && !dtype_size(a.bias_dtype))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: bias in fp32 or 16 bits (dtype %d)", what, a.bias_dtype);
  if (a.bias && (uintptr_t)a.bias % dtype_size(a.bias_dtype)) return set_error(ATMA_ERR_INVALID, "%s: misaligned bias", what);
  const int64_t tokens = (a.M + 15) / 16;
  const int64_t most = 65535;
  for (int64_t t = 0; t < tokens; t += most) {
    Fp4Args p = a;
    p.M = std::min(most * 16, a.M - t * 16);
    p.x = (const char*)a.x + t * 16 * a.ldx * 2;
    p.y = (char*)a.y + t * 16 * a.ldy * 2;
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((p.M + 15) / 16));
    auto launch = [&](auto zero) {
      using T = decltype(zero);
      if (gated) fp4_kernel<T, true><<<grid, 64, 0, (hipStream_t)stream>>>(p);
      else fp4_kernel<T, false><<<grid, 64, 0, (hipStream_t)stream>>>(p);
    };
    if (dtype == ATMA_BF16) launch(bf16{});
    else launch(f16{});
  }
  return check_launch(what);
}

}  // namespace atma

extern "C" int atma_linear_fp4(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* ws, int64_t ldws,
                               const void* bias, int bias_dtype, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                               int dtype, void* stream) {
  atma::Fp4Args a{x, ldx, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws, bias, bias_dtype, y, ldy, M, N, 0};
  return atma::linear_fp4("linear_fp4", false, a, K, dtype, stream);
}

extern "C" int atma_linear_gated_fp4(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* ws, int64_t ldws,
                                     const void* bias, int bias_dtype, void* y, int64_t ldy, int64_t M, int64_t H, int64_t K,
                                     int dtype, void* stream) {
  atma::Fp4Args a{x, ldx, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws, bias, bias_dtype, y, ldy, M, H, 0};
  return atma::linear_fp4("linear_gated_fp4", true, a, K, dtype, stream);
}
