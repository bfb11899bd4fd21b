// Quantizers to the 8-bit format of fp8.h: rows (activations, a scale for each 128 values of a row) and weights (a scale
// for each 128 x 128 block).  No reference counterpart.
//
// Both read each value once, keep it in registers through the reduction of its block's largest magnitude and write one
// byte for it, so they are bound by memory: 3 bytes a 16-bit value, 5 a 32-bit one.
#include <algorithm>

#include "fp8.h"

namespace atma {

// eight consecutive values as floats
template <typename T>
__device__ __forceinline__ void load8f(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else {
    const u32x4 u = *(const u32x4*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = elem16<T>(u, e);
  }
}

struct QuantArgs {
  const void* x;  // (M, K), row stride ldx
  int64_t ldx;
  uint8_t* data;  // (M, K), row stride ldd
  int64_t ldd;
  uint8_t* scale;  // (M, ceil(K / 128)), row stride lds
  int64_t lds;
  int64_t M;
  int K;
  int groups;  // 512-column groups a row
};

// A wave takes 512 columns of a row, 8 consecutive values a lane: a block is the 16 lanes of a DPP row, its maximum four lane
// exchanges (65,536 x 4,096 from bf16: 137 to 144 us, 5.6 to 5.9 TB/s, where a copy runs at 4.9)
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t m = item / a.groups;
  if (m >= a.M) return;
  const int c = (int)(item - m * a.groups) * 512 + lane * 8;
  float v[8] = {};
  if (c < a.K) load8f<T>((const T*)a.x + m * a.ldx + c, v);
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
  const int code = fp8_scale_code(row16_max(amax));
  if (c >= a.K) return;
  const float inv = fp8_inv_scale(code);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= inv;
  *(u32x2*)(a.data + m * a.ldd + c) = u32x2{fp8_pack4(v[0], v[1], v[2], v[3]), fp8_pack4(v[4], v[5], v[6], v[7])};
  if ((lane & 15) == 0) a.scale[m * a.lds + c / kFp8Block] = (uint8_t)code;
}

// A workgroup takes one 128 x 128 block: thread t the 8 columns 8 (t % 16) of rows t / 16, + 16, ..., all 64 values in
// registers through the maximum (8,192 x 1,024 from fp32: 7.5 us, 5.6 TB/s)
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(QuantArgs a) {
  __shared__ float part[4];
  const int t = threadIdx.x;
  const int c = (int)blockIdx.x * kFp8Block + 8 * (t & 15);
  const int64_t m0 = (int64_t)blockIdx.y * kFp8Block + (t >> 4);
  float v[8][8] = {};
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c < a.K && m0 + 16 * i < a.M) load8f<T>((const T*)a.x + (m0 + 16 * i) * a.ldx + c, v[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[i][e]));
  amax = wave_max(amax);
  if ((t & 63) == 0) part[t >> 6] = amax;
  __syncthreads();
  const int code = fp8_scale_code(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float inv = fp8_inv_scale(code);
  if (t == 0) a.scale[(int64_t)blockIdx.y * a.lds + blockIdx.x] = (uint8_t)code;
  if (c >= a.K) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (m0 + 16 * i < a.M) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= inv;
      *(u32x2*)(a.data + (m0 + 16 * i) * a.ldd + c) =
          u32x2{fp8_pack4(v[i][0], v[i][1], v[i][2], v[i][3]), fp8_pack4(v[i][4], v[i][5], v[i][6], v[i][7])};
    }
}

static int quantize(const char* what, bool weight, const void* x, int64_t ldx, void* data, int64_t ldd, void* scale,
                    int64_t lds, int64_t M, int64_t K, int dtype, void* stream) {
  const int size = dtype_size(dtype);
  if (!size) return set_error(ATMA_ERR_UNSUPPORTED, "%s: fp32 or 16-bit input (dtype %d)", what, dtype);
  if (M < 0 || K < 16 || K % 16 || K > (1 << 24) || M > 0x7fffffff)
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: K must be a multiple of 16 up to 2^24, M below 2^31 (M=%lld K=%lld)", what,
                     (long long)M, (long long)K);
  if (M == 0) return ATMA_OK;
  if (!x || !data || !scale) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  const int64_t nb = (K + kFp8Block - 1) / kFp8Block;
  if ((uintptr_t)x % 16 || (ldx * size) % 16 || ldx < K || (uintptr_t)data % 8 || ldd % 8 || ldd < K || lds < nb)
    return set_error(ATMA_ERR_INVALID, "%s: rows of x must be 16-byte aligned, rows of data 8-byte", what);
  QuantArgs a{x, ldx, (uint8_t*)data, ldd, (uint8_t*)scale, lds, M, (int)K, (int)((K + 511) / 512)};
  hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    if (weight) {
      const int64_t mb = (M + kFp8Block - 1) / kFp8Block;
      quantize_weight_kernel<T><<<dim3((unsigned)nb, (unsigned)mb), 256, 0, s>>>(a);
    } else {
      // a wave for each 512 columns of a row; a launch holds fewer than 2^32 threads, so what no one launch holds goes in
      // several (waves that stride over the rows instead cost 8% at 65,536 x 4,096)
      const int64_t rows = ((1 << 24) - 1) * 4ll / a.groups;
      for (int64_t m = 0; m < M; m += rows) {
        QuantArgs p = a;
        p.M = std::min(rows, M - m);
        p.x = (const T*)a.x + m * ldx;
        p.data += m * ldd;
        p.scale += m * lds;
        quantize_rows_kernel<T><<<dim3((unsigned)((p.M * a.groups + 3) / 4)), 256, 0, s>>>(p);
      }
    }
  };
  if (weight && (M + kFp8Block - 1) / kFp8Block > 65535)
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: at most %d rows", what, 65535 * kFp8Block);
  if (dtype == ATMA_BF16) launch(bf16{});
  else if (dtype == ATMA_F16) launch(f16{});
  else launch(float{});
  return check_launch(what);
}

}  // namespace atma

extern "C" int atma_quantize_fp8(const void* x, int64_t ldx, void* data, int64_t ldd, void* scale, int64_t lds,
                                 int64_t M, int64_t K, int dtype, void* stream) {
  return atma::quantize("quantize_fp8", false, x, ldx, data, ldd, scale, lds, M, K, dtype, stream);
}

extern "C" int atma_quantize_weight_fp8(const void* w, int64_t ldw, void* data, int64_t ldd, void* scale, int64_t lds,
                                        int64_t N, int64_t K, int dtype, void* stream) {
  return atma::quantize("quantize_weight_fp8", true, w, ldw, data, ldd, scale, lds, N, K, dtype, stream);
}
