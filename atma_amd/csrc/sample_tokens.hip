// Next-token sampling: temperature, top-k, top-p and min-p, from one given random number a row.  No counterpart in the
// reference beyond its temperature sampler (inference/layers/sampler.py:5-10).
//
// For a row x of V logits with temperature t > 0, w_i = exp((x_i - max x) / t).  The tokens stand in order of falling x, equal
// ones in the order of their indices, and each filter keeps a beginning of that order: top-k its first k; top-p the tokens
// before which less than p of the weight that top-k kept lies; min-p those with w_i >= m.  The answer is the first token, in
// index order, at which the sum of the kept weights exceeds u times their whole sum.
//
// No row is sorted: a beginning of the order is a value and, among the tokens that hold exactly it, a number of them.  The
// value is found by histograms of the values' order-preserving integers, 2,048 bins a level, of counts for top-k and of weights
// for top-p; the index among equal ones and the answer by sums over the waves' parts of the row, then inside one part.
//
// Weights are formed in fp64 and held as integers, multiples of 2^-43 of the largest: their sums are exact, so neither the
// order of the additions nor the number of threads changes a result, and a border is decided as in 64-bit arithmetic
// (with fp32 weights one row in a few thousand would answer its neighbour's token).  V <= 2^20 keeps every sum below 2^63.
#include <algorithm>

#include "common.h"

namespace atma {

struct SampleArgs {
  const void* logits;  // (rows, V), row stride ld
  int64_t ld;
  const float* uniform;      // (rows,)
  const float* temperature;  // (rows,), or null: t0 for every row; the filters likewise
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float t0, p0, m0;
  int k0;
  int64_t* ids;  // (rows,)
  int64_t rows;
  int V;
};

constexpr int kSampleBins = 2048;
constexpr int kSampleChunk = 512;  // logits of a wave at a time, 8 a lane
constexpr uint64_t kSampleOne = 1ull << 43;

// Values as integers in the values' order: -0 as +0, every NaN above +infinity; 0 stands for no logit at all
template <typename T>
struct SampleKey {
  static constexpr uint32_t kNan = 0xffffu;
  static __device__ __forceinline__ uint32_t of(uint32_t raw) {
    const uint32_t inf = __is_same(T, bf16) ? 0x7f80u : 0x7c00u;
    if ((raw & 0x7fffu) > inf) return kNan;
    if (raw == 0x8000u) raw = 0;
    return raw & 0x8000u ? raw ^ 0xffffu : raw | 0x8000u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return to_f32(__builtin_bit_cast(T, (uint16_t)(key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu)));
  }
};
template <>
struct SampleKey<float> {
  static constexpr uint32_t kNan = 0xffffffffu;
  static __device__ __forceinline__ uint32_t of(uint32_t raw) {
    if ((raw & 0x7fffffffu) > 0x7f800000u) return kNan;
    if (raw == 0x80000000u) raw = 0;
    return raw & 0x80000000u ? ~raw : raw | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
  }
};

__device__ __forceinline__ uint64_t wave_xor64(uint64_t x, int m) {
  return (uint64_t)__shfl_xor((unsigned long long)x, m, 64);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += wave_xor64(x, m);
  return x;
}
// The sum over this lane and the ones below it
__device__ __forceinline__ uint64_t wave_scan64(uint64_t x, int lane) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t y = (uint64_t)__shfl_up((unsigned long long)x, m, 64);
    if (lane >= m) x += y;
  }
  return x;
}

typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

// The keys of logits i .. i + 7, 0 past the end.  Rows start at any element: vector loads take any address
template <typename T>
__device__ __forceinline__ void sample_load8(const T* row, int i, int V, uint32_t* key) {
  if (i + 8 <= V) {
    if constexpr (sizeof(T) == 4) {
      const u32x4 a = *(const u32x4_at4*)(row + i), b = *(const u32x4_at4*)(row + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) key[e] = SampleKey<T>::of(a[e]), key[4 + e] = SampleKey<T>::of(b[e]);
    } else {
      const u32x4 a = *(const u32x4_at2*)(row + i);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        key[2 * e] = SampleKey<T>::of(a[e] & 0xffffu), key[2 * e + 1] = SampleKey<T>::of(a[e] >> 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      key[e] = 0;
      if (i + e < V) {
        if constexpr (sizeof(T) == 4) key[e] = SampleKey<T>::of(((const uint32_t*)row)[i + e]);
        else key[e] = SampleKey<T>::of(((const uint16_t*)row)[i + e]);
      }
    }
  }
}

// A row's workgroup: NW waves, each with a contiguous part of it
template <typename T, int NW>
struct Sampler {
  static constexpr int NT = 64 * NW, PER = kSampleBins / NT;
  struct Shared {
    unsigned long long bins[kSampleBins];
    unsigned long long part[NW];
    uint64_t found[3];
  };
  Shared* sh;
  const T* row;
  int V, lane, wave, first, last;  // the wave's part in chunks
  uint32_t top;                    // the largest key
  double xmax, inv_t;

  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int c = first; c < last; ++c) {
      const int i = c * kSampleChunk + 8 * lane;
      uint32_t key[8];
      sample_load8<T>(row, i, V, key);
#pragma unroll
      for (int e = 0; e < 8; ++e) f(i + e, key[e]);
    }
  }

  // (x - max) / t, 0 for every largest logit, whatever it is
  __device__ __forceinline__ double exponent(uint32_t key) const {
    return key == top ? 0.0 : ((double)SampleKey<T>::value(key) - xmax) * inv_t;
  }
  // below exp(-30.5) a weight rounds to 0 (a missing logit's key is that of a NaN: 0 too)
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    const double z = exponent(key);
    return z > -31.0 ? (uint64_t)(exp(z) * (double)kSampleOne + 0.5) : 0;
  }

  // Where the tokens in order first hold `target` (>= 1, at most the whole sum) of count(key): the key, what lies above it
  // and what tokens of that key hold together.  lo and hi bracket the keys of interest; no key below lo counts.
  template <typename F>
  __device__ __forceinline__ void select(uint32_t lo, uint32_t hi, uint64_t target, F count, uint32_t& at, uint64_t& above,
                                         uint64_t& held) {
    above = 0;
    while (true) {
      const int bits = 32 - __clz((int)(hi - lo));
      const int shift = bits > 11 ? bits - 11 : 0;
      for (int b = threadIdx.x; b < kSampleBins; b += NT) sh->bins[b] = 0;
      __syncthreads();
      each([&](int, uint32_t key) {
        if (key >= lo && key <= hi) {
          const uint64_t n = count(key);
          if (n) atomicAdd(&sh->bins[(hi - key) >> shift], (unsigned long long)n);
        }
      });
      __syncthreads();
      uint64_t mine = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) mine += sh->bins[PER * threadIdx.x + j];
      const uint64_t upto = wave_scan64(mine, lane);
      if (lane == 63) sh->part[wave] = upto;
      __syncthreads();
      uint64_t before = above + upto - mine;
      for (int q = 0; q < wave; ++q) before += sh->part[q];
      if (before < target && before + mine >= target) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint64_t n = sh->bins[PER * threadIdx.x + j];
          if (before < target && before + n >= target) {
            sh->found[0] = PER * threadIdx.x + j;
            sh->found[1] = before;
            sh->found[2] = n;
          }
          before += n;
        }
      }
      __syncthreads();
      const uint32_t b = (uint32_t)sh->found[0];
      above = sh->found[1];
      held = sh->found[2];
      __syncthreads();
      hi -= b << shift;
      if (shift == 0) {
        at = hi;
        return;
      }
      const uint32_t span = (1u << shift) - 1;
      lo = hi - lo > span ? hi - span : lo;
    }
  }

  __device__ __forceinline__ uint64_t block_sum(uint64_t x) {
    x = wave_sum64(x);
    if (lane == 0) sh->part[wave] = x;
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (int q = 0; q < NW; ++q) sum += sh->part[q];
    __syncthreads();
    return sum;
  }

  // The first index at which the sum of amount(index, key) passes target; total: the whole sum.  target(total) < total
  template <typename F, typename G>
  __device__ __forceinline__ int find(F amount, G target) {
    uint64_t mine = 0;
    each([&](int i, uint32_t key) { mine += amount(i, key); });
    mine = wave_sum64(mine);
    if (lane == 0) sh->part[wave] = mine;
    __syncthreads();
    uint64_t sum = 0, before = 0;
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      if (q == wave) before = sum;
      sum += sh->part[q];
    }
    const uint64_t aim = target(sum);
    if (before <= aim && aim < before + mine) {  // one wave, all of it
      for (int c = first; c < last; ++c) {
        const int i = c * kSampleChunk + 8 * lane;
        uint32_t key[8];
        sample_load8<T>(row, i, V, key);
        uint64_t own = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own += amount(i + e, key[e]);
        const uint64_t upto = wave_scan64(own, lane);
        uint64_t at = before + upto - own;
        if (at <= aim && aim < at + own) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint64_t n = amount(i + e, key[e]);
            if (at <= aim && aim < at + n) sh->found[0] = (uint64_t)(i + e);
            at += n;
          }
        }
        before += (uint64_t)__shfl((unsigned long long)upto, 63, 64);
        if (aim < before) break;
      }
    }
    __syncthreads();
    const int i = (int)sh->found[0];
    __syncthreads();
    return i;
  }
};

template <typename T, int NW>
__global__ void __launch_bounds__(64 * NW) sample_tokens_kernel(SampleArgs a) {
  using S = Sampler<T, NW>;
  __shared__ typename S::Shared shared;
  S s;
  s.sh = &shared;
  s.V = a.V;
  s.lane = threadIdx.x & 63;
  s.wave = threadIdx.x >> 6;
  const int chunks = (a.V + kSampleChunk - 1) / kSampleChunk, each = (chunks + NW - 1) / NW;
  s.first = min(s.wave * each, chunks);
  s.last = min(s.first + each, chunks);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    s.row = (const T*)a.logits + r * a.ld;
    // the largest logit, at its lowest index, and the smallest
    uint64_t best = 0;
    uint32_t least = 0xffffffffu;
    s.each([&](int i, uint32_t key) {
      const uint64_t v = (uint64_t)key << 32 | (uint32_t)~i;
      best = v > best ? v : best;
      least = key && key < least ? key : least;
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const uint64_t v = wave_xor64(best, m);
      best = v > best ? v : best;
      least = min(least, (uint32_t)__shfl_xor((int)least, m, 64));
    }
    if (s.lane == 0) shared.bins[2 * s.wave] = best, shared.bins[2 * s.wave + 1] = least;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      best = max(best, (uint64_t)shared.bins[2 * q]);
      least = min(least, (uint32_t)shared.bins[2 * q + 1]);
    }
    __syncthreads();
    s.top = (uint32_t)(best >> 32);
    int answer = (int)~(uint32_t)best;
    const float t = a.temperature ? a.temperature[r] : a.t0;
    if (t > 0.f && s.top != SampleKey<T>::kNan) {  // (else the largest logit; a NaN is above all, as in torch's argmax)
      s.xmax = (double)SampleKey<T>::value(s.top);
      s.inv_t = 1.0 / (double)t;
      const int k = a.top_k ? a.top_k[r] : a.k0;
      const float p = a.top_p ? a.top_p[r] : a.p0, m = a.min_p ? a.min_p[r] : a.m0;
      // a beginning of the order: every token above `at`, and of those that hold it the first `n`
      uint32_t at = 0;
      uint64_t n = 0, above, held;
      bool cut = false;  // not all of them
      if (k > 0 && k < a.V) {
        s.select(least, s.top, (uint64_t)k, [](uint32_t) { return (uint64_t)1; }, at, above, held);
        n = (uint64_t)k - above;
        cut = n < held;
      }
      if (p < 1.f) {  // (NaN: no filter)
        uint64_t sum = 0;
        const uint32_t kk = at;
        s.each([&](int, uint32_t key) { sum += key > kk ? s.weight(key) : 0; });
        sum = s.block_sum(sum);
        const uint64_t one = kk ? s.weight(kk) : 0;
        sum += n * one;
        const double want = (double)p * (double)sum;
        const uint64_t target = min(max((uint64_t)(want > 0.0 ? ceil(want) : 1.0), (uint64_t)1), sum);
        uint32_t pk;
        s.select(kk ? kk : least, s.top, target, [&](uint32_t key) { return s.weight(key); }, pk, above, held);
        const uint64_t w = s.weight(pk), take = (target - above + w - 1) / w, ties = held / w;
        if (pk != kk || take < n) {
          cut = (pk == kk && cut) || take < ties;
          n = take;
        }
        at = pk;
      }
      int end = a.V;
      if (cut) end = s.find([&](int, uint32_t key) { return (uint64_t)(key == at); }, [&](uint64_t) { return n - 1; });
      const double floor_z = m > 0.f ? log((double)fminf(m, 1.f)) : -INFINITY;
      const float u = a.uniform[r];
      answer = s.find(
          [&](int i, uint32_t key) {
            const bool kept = key > at || (key == at && i <= end);
            return kept && s.exponent(key) >= floor_z ? s.weight(key) : (uint64_t)0;
          },
          [&](uint64_t sum) {
            const double f = u > 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
            return (uint64_t)(f * (double)sum);
          });
    }
    if (threadIdx.x == 0) a.ids[r] = answer;
  }
}

}  // namespace atma

extern "C" int atma_sample_tokens(const void* logits, int64_t ld, const float* uniform, const float* temperature, float t0,
                                  const int32_t* top_k, int k0, const float* top_p, float p0, const float* min_p, float m0,
                                  int64_t* ids, int64_t rows, int64_t V, int dtype, void* stream) {
  using namespace atma;
  const char* what = "sample_tokens";
  if (!dtype_size(dtype)) return set_error(ATMA_ERR_UNSUPPORTED, "%s: fp32 or 16-bit logits (dtype %d)", what, dtype);
  if (rows < 0 || V < 1 || V > (1 << 20))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: 1 to 2^20 logits a row (rows=%lld V=%lld)", what, (long long)rows, (long long)V);
  if (rows == 0) return ATMA_OK;
  if (!logits || !uniform || !ids) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)logits % dtype_size(dtype)) return set_error(ATMA_ERR_INVALID, "%s: misaligned logits", what);
  if (rows > 1 && ld < V && ld != 0) return set_error(ATMA_ERR_INVALID, "%s: rows overlap", what);
  SampleArgs a{logits, ld, uniform, temperature, top_k, top_p, min_p, t0, p0, m0, k0, ids, rows, (int)V};
  const unsigned grid = (unsigned)std::min<int64_t>(rows, 1 << 20);
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    if (V <= 8192) sample_tokens_kernel<T, 4><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else sample_tokens_kernel<T, 16><<<grid, 1024, 0, (hipStream_t)stream>>>(a);
  };
  if (dtype == ATMA_BF16) launch(bf16{});
  else if (dtype == ATMA_F16) launch(f16{});
  else launch(float{});
  return check_launch(what);
}
