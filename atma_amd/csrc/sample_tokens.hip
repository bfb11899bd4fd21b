// Next-token sampling: temperature, top-k, top-p and min-p, from one given random number a row.  No counterpart in the
// reference beyond its temperature sampler (inference/layers/sampler.py:5-10).
//
// For a row x of V logits with temperature t > 0, w_i = exp((x_i - max x) / t).  The tokens stand in order of falling x, equal
// ones in the order of their indices, and each filter keeps a beginning of that order: top-k its first k; top-p the tokens
// before which less than p of the weight that top-k kept lies; min-p those with w_i >= m.  The answer is the first token, in
// index order, at which the sum of the kept weights exceeds u times their whole sum.
//
// No row is sorted.  One pass finds the largest logit, a second one counts the tokens (top-k) and adds up their weights (top-p) in
// bins of equal width below it; a filter's border lies in one bin, whose tokens, a hundred or so, are gathered and ranked, each
// against all others.  That gives the last token kept, a value and an index.  A last pass sums the kept weights of each wave's part
// of the row, and the wave in whose part the answer lies finds it.  Where a bin holds more than fits the list (many equal logits)
// the border's value is found by histograms of the values' order-preserving integers, 2,048 bins a level, then the index.
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

constexpr int kSampleBins = 2048;   // of a level of the exact search
constexpr int kSampleChunk = 512;   // logits of a wave at a time, 8 a lane
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

// Logits i .. i + 7 of a row as they lie in memory.  Rows start at any element: vector loads take any address
template <typename T>
struct SampleRaw {
  u32x4 v[sizeof(T) == 4 ? 2 : 1];
  __device__ __forceinline__ void load(const T* row, int i, int V) {
    if (i + 8 <= V) {
      if constexpr (sizeof(T) == 4) v[0] = *(const u32x4_at4*)(row + i), v[1] = *(const u32x4_at4*)(row + i + 4);
      else v[0] = *(const u32x4_at2*)(row + i);
    } else {
      // the end of a row: nothing behind it is read
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 4) {
          v[e >> 2][e & 3] = i + e < V ? ((const uint32_t*)row)[i + e] : 0u;
        } else {
          const uint32_t u = i + e < V ? ((const uint16_t*)row)[i + e] : 0u;
          if (e & 1) v[0][e >> 1] |= u << 16;
          else v[0][e >> 1] = u;
        }
      }
    }
  }
  __device__ __forceinline__ uint32_t raw(int e) const {
    if constexpr (sizeof(T) == 4) return v[e >> 2][e & 3];
    else return (v[0][e >> 1] >> (16 * (e & 1))) & 0xffffu;
  }
};

// A token in the order: its key, then the lower index first
__device__ __forceinline__ uint64_t sample_order(uint32_t key, int i) { return (uint64_t)key << 32 | (uint32_t)~i; }

// A row's workgroup: NW waves, each with a contiguous part of it
template <typename T, int NW>
struct Sampler {
  static constexpr int NT = 64 * NW, PER = kSampleBins / NT;
  static constexpr int B = NW >= 8 ? 4096 : 1024, BPER = B / NT, LIST = NT;
  struct Shared {
    unsigned long long mass[B > kSampleBins ? B : kSampleBins];
    uint32_t count[B];
    uint64_t key[LIST], weight[LIST];  // the tokens of one bin
    double power[256];                 // 2^(j / 256)
    unsigned long long part[NW];
    uint64_t found[3];
    unsigned long long last, sum;
    uint32_t n;
  };
  Shared* sh;
  const T* row;
  int V, lane, wave, first, last;  // the wave's part in chunks
  uint32_t top, least;             // the largest and the smallest key
  float xtop, width;               // the largest logit; bins a unit of logits
  double xmax, c;                  // the same; log2(e) / temperature

  // f(index, key) for every logit of the wave's part, loads a chunk ahead
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    SampleRaw<T> next;
    if (first < last) next.load(row, first * kSampleChunk + 8 * lane, V);
    for (int q = first; q < last; ++q) {
      const SampleRaw<T> now = next;
      const int i = q * kSampleChunk + 8 * lane;
      if (q + 1 < last) next.load(row, i + kSampleChunk, V);
      if ((q + 1) * kSampleChunk <= V) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f(i + e, SampleKey<T>::of(now.raw(e)));
          if (e & 1) __builtin_amdgcn_sched_barrier(0);  // (eight exponentials side by side take more registers than there are)
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f(i + e, i + e < V ? SampleKey<T>::of(now.raw(e)) : 0u);
      }
    }
  }

  // 2^43 exp((x - max) / t), rounded; 2^43 for every largest logit, whatever it is.  2^y for y = n + j / 256 + r: a table's value
  // times the Taylor polynomial of 2^r, |r| <= 1 / 512, of degree 4 (4e-17 off); the sums with powers of two round to
  // multiples of 1 / 256 and to whole numbers.  (A missing logit's key is that of a NaN: 0)
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    const double y = fmax(fma((double)SampleKey<T>::value(k) - xmax, c, 43.0), -3.0);
    const double s = y + 0x1.8p44, r = y - (s - 0x1.8p44);
    const int j = (int)(uint32_t)__builtin_bit_cast(uint64_t, s);
    double p = fma(r, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0c0p-5);
    p = fma(p, r, 0x1.ebfbdff82c58fp-3);
    p = fma(p, r, 0x1.62e42fefa39efp-1);
    const double b = sh->power[j & 255];
    const double w = __builtin_amdgcn_ldexp(fma(b, p * r, b), j >> 8) + 0x1p52;
    const uint64_t u = __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
    return k == top ? kSampleOne : u;
  }

  // A logit's bin: equal widths below the largest; what has no weight lies in the last one, which holds nothing else
  __device__ __forceinline__ int bin(uint32_t k) const {
    const int b = (int)fminf((xtop - SampleKey<T>::value(k)) * width, (float)(B - 1));
    return k == top ? 0 : b;
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

  // The bin at which the bins' sums first hold `target` (>= 1, at most the whole sum): what lies above it and what it holds
  template <int N, typename A>
  __device__ __forceinline__ int find_bin(const A* bins, uint64_t above, uint64_t target, uint64_t& before, uint64_t& held) {
    uint64_t v[N], mine = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) mine += v[j] = bins[N * threadIdx.x + j];
    const uint64_t upto = wave_scan64(mine, lane);
    if (lane == 63) sh->part[wave] = upto;
    __syncthreads();
    uint64_t at = above + upto - mine;
    for (int q = 0; q < wave; ++q) at += sh->part[q];
    if (at < target && at + mine >= target) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (at < target && at + v[j] >= target) {
          sh->found[0] = N * threadIdx.x + j;
          sh->found[1] = at;
          sh->found[2] = v[j];
        }
        at += v[j];
      }
    }
    __syncthreads();
    const int b = (int)sh->found[0];
    before = sh->found[1];
    held = sh->found[2];
    __syncthreads();
    return b;
  }

  // The tokens of bin b into the list
  __device__ __forceinline__ int gather(int b) {
    if (threadIdx.x == 0) sh->n = 0;
    __syncthreads();
    each([&](int i, uint32_t k) {
      if (k && bin(k) == b) {
        const uint32_t at = atomicAdd(&sh->n, 1u);
        if (at < (uint32_t)LIST) sh->key[at] = sample_order(k, i), sh->weight[at] = weight(k);
      }
    });
    __syncthreads();
    return (int)sh->n;
  }

  // The last token of the list, in order, that keep(tokens before it in the list, their weight) keeps, at least one; sum: the kept
  // tokens' weight
  template <typename F>
  __device__ __forceinline__ uint64_t cut(int n, F keep, uint64_t& sum) {
    if (threadIdx.x == 0) sh->last = ~0ull, sh->sum = 0;
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const uint64_t k = sh->key[threadIdx.x];
      uint32_t rank = 0;
      uint64_t before = 0;
      for (int j = 0; j < n; ++j)
        if (sh->key[j] > k) ++rank, before += sh->weight[j];
      if (keep(rank, before)) {
        atomicMin(&sh->last, (unsigned long long)k);
        atomicAdd(&sh->sum, (unsigned long long)sh->weight[threadIdx.x]);
      }
    }
    __syncthreads();
    const uint64_t k = sh->last;
    sum = sh->sum;
    __syncthreads();
    return k;
  }

  // The exact search: where the tokens in order, those from `from` on left out, first hold `target` (>= 1, at most the whole sum)
  // of amount(key).  Returns the last token needed
  template <typename F>
  __device__ __forceinline__ uint64_t search(uint64_t from, uint64_t target, F amount) {
    uint32_t hi = top, lo = max(least, (uint32_t)(from >> 32));
    uint64_t above = 0, held;
    while (true) {
      const int bits = 32 - __clz((int)(hi - lo));
      const int shift = bits > 11 ? bits - 11 : 0;
      for (int b = threadIdx.x; b < kSampleBins; b += NT) sh->mass[b] = 0;
      __syncthreads();
      each([&](int, uint32_t k) {
        if (k >= lo && k <= hi) {
          const uint64_t n = amount(k);
          if (n) atomicAdd(&sh->mass[(hi - k) >> shift], (unsigned long long)n);
        }
      });
      __syncthreads();
      hi -= (uint32_t)find_bin<PER>(sh->mass, above, target, above, held) << shift;
      if (shift == 0) break;
      const uint32_t span = (1u << shift) - 1;
      lo = hi - lo > span ? hi - span : lo;
    }
    // of the tokens that hold exactly this value the first so many
    const uint64_t one = amount(hi), n = (target - above + one - 1) / one;
    if (n * one >= held) return sample_order(hi, V - 1);
    return sample_order(hi, find([&](int, uint32_t k) { return (uint64_t)(k == hi); }, [&](uint64_t) { return n - 1; }));
  }

  // The first index at which the sum of amount(index, key) passes target(the whole sum), which is below it
  template <typename F, typename G>
  __device__ __forceinline__ int find(F amount, G target) {
    uint64_t mine = 0;
    each([&](int i, uint32_t k) { mine += amount(i, k); });
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
      for (int q = first; q < last; ++q) {
        const int i = q * kSampleChunk + 8 * lane;
        SampleRaw<T> now;
        now.load(row, i, V);
        uint64_t n[8], own = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own += n[e] = amount(i + e, i + e < V ? SampleKey<T>::of(now.raw(e)) : 0u);
        const uint64_t upto = wave_scan64(own, lane);
        uint64_t at = before + upto - own;
        if (at <= aim && aim < at + own) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (at <= aim && aim < at + n[e]) sh->found[0] = (uint64_t)(i + e);
            at += n[e];
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

  // The last token that top-k and top-p keep (0: every one)
  __device__ __forceinline__ uint64_t border(int k, float p) {
    const bool by_count = k > 0 && k < V, by_mass = p < 1.f;  // (a NaN is no filter)
    if (!by_count && !by_mass) return 0;
    for (int b = threadIdx.x; b < B; b += NT) sh->mass[b] = 0, sh->count[b] = 0;
    __syncthreads();
    each([&](int, uint32_t key) {
      if (!key) return;
      const int b = bin(key);
      if (by_count) atomicAdd(&sh->count[b], 1u);
      if (by_mass) atomicAdd(&sh->mass[b], (unsigned long long)weight(key));
    });
    __syncthreads();
    uint64_t keep = 0, above, held, total = 0;
    bool slow = false;
    int listed = -1;  // the bin in the list
    if (by_count) {
      const int b = find_bin<BPER>(sh->count, 0, (uint64_t)k, above, held);
      if (b < B - 1) {  // (else every token with a weight is among them)
        slow = held > LIST;
        if (!slow) {
          listed = b;
          keep = cut(gather(b), [&](uint32_t rank, uint64_t) { return above + rank < (uint64_t)k; }, total);
        }
      }
      if (slow) keep = search(0, (uint64_t)k, [](uint32_t) { return (uint64_t)1; });
    }
    if (!by_mass) return keep;
    if (slow) {
      uint64_t mine = 0;
      each([&](int i, uint32_t key) { mine += sample_order(key, i) >= keep ? weight(key) : 0; });
      total = block_sum(mine);
    } else {
      // the bins above the list's, and what of it is kept
      uint64_t mine = 0;
#pragma unroll
      for (int j = 0; j < BPER; ++j)
        if (listed < 0 || (int)(BPER * threadIdx.x + j) < listed) mine += sh->mass[BPER * threadIdx.x + j];
      total += block_sum(mine);
    }
    const double want = (double)p * (double)total;
    const uint64_t target = min(max((uint64_t)(want > 0.0 ? ceil(want) : 1.0), (uint64_t)1), total);
    if (!slow) {
      const int b = find_bin<BPER>(sh->mass, 0, target, above, held);
      if (b != listed) {
        const int n = gather(b);
        slow = n > LIST;
      }
      if (!slow)
        return max(keep, cut((int)min(sh->n, (uint32_t)LIST), [&](uint32_t, uint64_t before) { return above + before < target; }, held));
    }
    return max(keep, search(keep, target, [&](uint32_t key) { return weight(key); }));
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
  for (int j = threadIdx.x; j < 256; j += S::NT) shared.power[j] = exp2(j / 256.0);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    s.row = (const T*)a.logits + r * a.ld;
    // the largest logit, at its lowest index, and the smallest
    uint64_t best = 0;
    uint32_t least = 0xffffffffu;
    s.each([&](int i, uint32_t key) {
      const uint64_t v = sample_order(key, i);
      best = v > best ? v : best;
      least = key && key < least ? key : least;
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const uint64_t v = wave_xor64(best, m);
      best = v > best ? v : best;
      least = min(least, (uint32_t)__shfl_xor((int)least, m, 64));
    }
    if (s.lane == 0) shared.mass[2 * s.wave] = best, shared.mass[2 * s.wave + 1] = least;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      best = max(best, (uint64_t)shared.mass[2 * q]);
      least = min(least, (uint32_t)shared.mass[2 * q + 1]);
    }
    __syncthreads();
    s.top = (uint32_t)(best >> 32);
    s.least = least;
    int answer = (int)~(uint32_t)best;
    const float t = a.temperature ? a.temperature[r] : a.t0;
    if (t > 0.f && s.top != SampleKey<T>::kNan) {  // (else the largest logit; a NaN is above all, as in torch's argmax)
      s.xtop = SampleKey<T>::value(s.top);
      s.xmax = (double)s.xtop;
      s.c = 1.4426950408889634 / (double)t;
      // every logit above the last bin, but what lies 31 temperatures below the largest
      s.width = (float)(S::B - 1) / fminf((s.xtop - SampleKey<T>::value(least)) * 1.001f, 31.f * t);
      if (!(s.width > 0.f && s.width < 3e38f)) s.width = 0.f;
      const uint64_t keep = s.border(a.top_k ? a.top_k[r] : a.k0, a.top_p ? a.top_p[r] : a.p0);
      const float m = a.min_p ? a.min_p[r] : a.m0, u = a.uniform[r];
      const double least_x = m >= 1.f ? s.xmax : m > 0.f ? s.xmax + (double)t * log((double)m) : -INFINITY;
      answer = s.find(
          [&](int i, uint32_t key) {
            const bool kept = key && sample_order(key, i) >= keep && !((double)SampleKey<T>::value(key) < least_x);
            return kept ? s.weight(key) : (uint64_t)0;
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
