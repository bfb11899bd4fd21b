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
// (with fp32 weights one row in a few thousand would answer its neighbour's token).  V <= 2^20 keeps every sum at 2^63 or
// below, in unsigned 64-bit integers.
//
// What bounds it is a CU's work on a row: two passes that form a weight for every logit, some 190 cycles for 64 of them.  512 rows of 50,304
// fp32 logits with top-p take 117 us, one in one workgroup 43, shared by 13 of them 23 to 24.
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
  int V;
  uint8_t* held;  // of few long rows: their workspace, WideRow's arrays for each
  int parts;
};

constexpr int kSampleBins = 2048;   // of a level of the exact search
constexpr int kSampleChunk = 512;   // logits of a wave at a time, 8 a lane
constexpr uint64_t kSampleOne = 1ull << 43;

// Values as integers in the values' order, -0 as +0
template <typename T>
struct SampleKey {
  static __device__ __forceinline__ uint32_t of_value(float x) {
    uint32_t raw = __builtin_bit_cast(uint16_t, from_f32<T>(x));
    if (raw == 0x8000u) raw = 0;
    return raw & 0x8000u ? raw ^ 0xffffu : raw | 0x8000u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return to_f32(__builtin_bit_cast(T, (uint16_t)(key & 0x8000u ? key & 0x7fffu : key ^ 0xffffu)));
  }
};
template <>
struct SampleKey<float> {
  static __device__ __forceinline__ uint32_t of_value(float x) {
    uint32_t raw = __builtin_bit_cast(uint32_t, x);
    if (raw == 0x80000000u) raw = 0;
    return raw & 0x80000000u ? ~raw : raw | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
  }
};

// The sum over this lane and the ones below it: lane exchanges inside rows of 16, then the rows' last lanes (no LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_add64(uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
  return x + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t row_scan64(uint64_t x) {
  x = dpp_add64<0x111, 0xF>(x);  // row_shr:1, 2, 4, 8
  x = dpp_add64<0x112, 0xF>(x);
  x = dpp_add64<0x114, 0xF>(x);
  return dpp_add64<0x118, 0xF>(x);
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t x) {
  x = row_scan64(x);
  x = dpp_add64<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  return dpp_add64<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t row_scan32(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan32(uint32_t x) {
  x = row_scan32(x);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_or32(uint32_t x) {
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint32_t lane32(uint32_t x, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)x, l); }
__device__ __forceinline__ uint64_t lane64(uint64_t x, int l) {
  return (uint64_t)lane32((uint32_t)(x >> 32), l) << 32 | lane32((uint32_t)x, l);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) { return wave_scan32(x); }
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) { return wave_scan64(x); }
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int l) { return lane32(x, l); }
__device__ __forceinline__ uint64_t lane_of(uint64_t x, int l) { return lane64(x, l); }
__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) { return lane64(wave_scan64(x), 63); }

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
  __device__ __forceinline__ float value(int e) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u = v[e >> 2][e & 3];  // (a bit cast of the element itself takes the vector's first)
      return __builtin_bit_cast(float, u);
    } else {
      return elem16<T>(v[0], e);
    }
  }
};

// 2^y for y = n + j / 256 + r: a table's value times the Taylor polynomial of 2^r, |r| <= 1 / 512, of degree 4 (4e-17 off); the sum
// with a power of two rounds to multiples of 1 / 256
__device__ __forceinline__ double sample_power(double y, const double* power) {
  const double s = y + 0x1.8p44, r = y - (s - 0x1.8p44);
  const int j = (int)(uint32_t)__builtin_bit_cast(uint64_t, s);
  double p = fma(r, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0bfp-5);
  p = fma(p, r, 0x1.ebfbdff82c58ep-3);
  p = fma(p, r, 0x1.62e42fefa39efp-1);
  const double b = power[j & 255];
  return __builtin_amdgcn_ldexp(fma(b, p * r, b), j >> 8);
}
// A number of [0, 2^51] rounded to the nearest integer
__device__ __forceinline__ uint64_t whole64(double w) {
  return __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull;
}
// 2^43 exp((x - max) / t), rounded, for c = log2(e) / t (NaN: 0)
__device__ __forceinline__ uint64_t sample_weight(double x, double xmax, double c, const double* power) {
  return whole64(sample_power(fmax(fma(x - xmax, c, 43.0), -3.0), power));
}

// A token in the order: its key, then the lower index first
__device__ __forceinline__ uint64_t sample_order(uint32_t key, int i) { return (uint64_t)key << 32 | (uint32_t)~i; }

// A row's workgroup: NW waves, each with a contiguous part of it.  Passes work on the values themselves (no row with a NaN comes
// past the first one): a missing logit, behind the row's end, reads as NaN, which no comparison keeps and which has no weight
template <typename T, int NW, int BINS = NW >= 16 ? 4096 : 1024, int LISTED = 64 * NW>
struct Sampler {
  typedef T Type;
  static constexpr int NT = 64 * NW, PER = kSampleBins / NT;
  static constexpr int B = BINS, BPER = B / NT, LIST = LISTED;
  struct Shared {
    unsigned long long mass[B > kSampleBins ? B : kSampleBins];
    uint32_t count[B];
    uint64_t key[LIST], weight[LIST];  // the tokens of one bin
    double power[256];                 // 2^(j / 256)
    unsigned long long part[NW];
    uint64_t found[3];
    unsigned long long last, sum;
    float top[NW], least[NW];
    uint32_t n, first;
  };
  Shared* sh;
  const T* row;
  int V, lane, wave, first, last;  // the wave's part in chunks
  float top, least, width;         // the largest and the smallest logit; bins a unit of logits
  double c;                        // log2(e) / temperature

  // A row's chunks from `from` to before `to`, among the waves
  __device__ __forceinline__ void start(const SampleArgs& a, int64_t r, int from, int to) {
    V = a.V;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int each = (to - from + NW - 1) / NW;
    first = min(from + wave * each, to);
    last = min(first + each, to);
    row = (const T*)a.logits + r * a.ld;
  }

  // f(index, value) for every logit of the wave's part, done(chunk) behind each chunk; loads a chunk ahead
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each(f, [](int) {});
  }
  template <typename F, typename D>
  __device__ __forceinline__ void each(F f, D done) const {
    SampleRaw<T> next;
    if (first < last) next.load(row, first * kSampleChunk + 8 * lane, V);
#pragma unroll 1
    for (int q = first; q < last; ++q) {
      const SampleRaw<T> now = next;
      const int i = q * kSampleChunk + 8 * lane;
      if (q + 1 < last) next.load(row, i + kSampleChunk, V);
      const bool whole = (q + 1) * kSampleChunk <= V;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = now.value(e);
        f(i + e, whole || i + e < V ? x : __builtin_nanf(""));
        if (e & 1) __builtin_amdgcn_sched_barrier(0);  // (eight exponentials side by side take more registers than there are)
      }
      done(q);
    }
  }

  // 2^43 for every largest logit, whatever it is
  __device__ __forceinline__ uint64_t weight(float x) const {
    const uint64_t w = sample_weight((double)x, (double)top, c, sh->power);
    return x == top ? kSampleOne : w;
  }

  // A logit's bin: equal widths below the largest; what has no weight lies in the last one, which holds nothing else
  __device__ __forceinline__ int bin(float x) const {
    const int b = (int)fminf((top - x) * width, (float)(B - 1));
    return x == top ? 0 : b;
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
    const uint64_t upto = wave_scan64(mine);
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
    each([&](int i, float x) {
      if (bin(x) == b && x == x) {
        const uint32_t at = atomicAdd(&sh->n, 1u);
        if (at < (uint32_t)LIST) sh->key[at] = sample_order(SampleKey<T>::of_value(x), i), sh->weight[at] = weight(x);
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
    for (int own = threadIdx.x; own < n; own += NT) {
      const uint64_t k = sh->key[own];
      uint32_t rank = 0;
      uint64_t before = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const bool above = sh->key[j] > k;
        rank += above;
        before += above ? sh->weight[j] : 0;
      }
      if (keep(rank, before)) {
        atomicMin(&sh->last, (unsigned long long)k);
        atomicAdd(&sh->sum, (unsigned long long)sh->weight[own]);
      }
    }
    __syncthreads();
    const uint64_t k = sh->last;
    sum = sh->sum;
    __syncthreads();
    return k;
  }

  // The exact search: where the tokens in order, those from `from` on left out, first hold `target` (>= 1, at most the whole sum)
  // of amount(value).  Returns the last token needed
  template <typename F>
  __device__ __forceinline__ uint64_t search(uint64_t from, uint64_t target, F amount) {
    uint32_t hi = SampleKey<T>::of_value(top), lo = max(SampleKey<T>::of_value(least), (uint32_t)(from >> 32));
    uint64_t above = 0, held;
    while (true) {
      const int bits = 32 - __clz((int)(hi - lo));
      const int shift = bits > 11 ? bits - 11 : 0;
      for (int b = threadIdx.x; b < kSampleBins; b += NT) sh->mass[b] = 0;
      __syncthreads();
      each([&](int, float x) {
        const uint32_t k = SampleKey<T>::of_value(x);
        if (k >= lo && k <= hi && x == x) {
          const uint64_t n = amount(x);
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
    const float at = SampleKey<T>::value(hi);
    const uint64_t one = amount(at), n = (target - above + one - 1) / one;
    if (n * one >= held) return sample_order(hi, V - 1);
    return sample_order(hi, find([&](int, float x) { return (uint64_t)(x == at); }, [&](uint64_t) { return n - 1; }));
  }

  // The first index at which the sum of amount(index, value) passes target(the whole sum), which is below it
  template <typename F, typename G>
  __device__ __forceinline__ int find(F amount, G target) {
    uint64_t own = 0;
    static_assert(sizeof(Shared::mass) >= 8 * ((1 << 20) / kSampleChunk), "a chunk's sum each: the bins are read");
    each([&](int i, float x) { own += amount(i, x); },
         [&](int q) {
           own = wave_sum64(own);
           if (lane == 0) sh->mass[q] = own;
           own = 0;
         });
    return find_in_chunks(amount, target);
  }
  // The same with every chunk's sum in `mass`
  template <typename F, typename G>
  __device__ __forceinline__ int find_in_chunks(F amount, G target) {
    __syncthreads();
    uint64_t mine = 0;
#pragma unroll 1
    for (int q = first; q < last; q += 64) mine += wave_sum64(q + lane < last ? sh->mass[q + lane] : 0);
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
      int q = first;
#pragma unroll 1
      for (;; q += 64) {
        const uint64_t v = q + lane < last ? sh->mass[q + lane] : 0, upto = before + wave_scan64(v);
        const uint64_t there = __ballot(aim < upto);
        if (there) {
          const int l = __builtin_ctzll(there);
          q += l;
          before = lane64(upto - v, l);
          break;
        }
        before = lane64(upto, 63);
      }
      const int i = q * kSampleChunk + 8 * lane;
      SampleRaw<T> now;
      now.load(row, i, V);
      uint64_t n[8], its = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) its += n[e] = amount(i + e, i + e < V ? now.value(e) : __builtin_nanf(""));
      uint64_t at = before + wave_scan64(its) - its;
      if (at <= aim && aim < at + its) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (at <= aim && aim < at + n[e]) sh->found[0] = (uint64_t)(i + e);
          at += n[e];
        }
      }
    }
    __syncthreads();
    const int i = (int)sh->found[0];
    __syncthreads();
    return i;
  }

  // The tokens up to a last one in order (0: every one)
  struct Kept {
    float at;
    int index;
    __device__ __forceinline__ explicit Kept(uint64_t last)
        : at(last ? SampleKey<T>::value((uint32_t)(last >> 32)) : -INFINITY), index(last ? (int)~(uint32_t)last : 0x7fffffff) {}
    __device__ __forceinline__ bool operator()(int i, float x) const { return x > at || (x == at && i <= index); }
  };

  // The last token that top-k and top-p keep (0: every one)
  __device__ __forceinline__ uint64_t border(int k, float p) {
    const bool by_count = k > 0 && k < V, by_mass = p < 1.f;  // (a NaN is no filter)
    if (!by_count && !by_mass) return 0;
    for (int b = threadIdx.x; b < B; b += NT) sh->mass[b] = 0, sh->count[b] = 0;
    __syncthreads();
    each([&](int, float x) {  // (a missing one is counted in the last bin, where it changes nothing)
      const int b = bin(x);
      if (by_count) atomicAdd(&sh->count[b], 1u);
      if (by_mass) atomicAdd(&sh->mass[b], (unsigned long long)weight(x));
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
      if (slow) keep = search(0, (uint64_t)k, [](float) { return (uint64_t)1; });
    }
    if (!by_mass) return keep;
    if (slow) {
      uint64_t mine = 0;
      const Kept kept(keep);
      each([&](int i, float x) { mine += kept(i, x) ? weight(x) : 0; });
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
    return max(keep, search(keep, target, [&](float x) { return weight(x); }));
  }
};

// The answer of row r, whose parts s has
template <typename S>
__device__ __forceinline__ int sample_row(S& s, const SampleArgs& a, int64_t r) {
  typename S::Shared& sh = *s.sh;
  // ---- the largest logit and the smallest, and whether there is a NaN
  float top = -INFINITY, least = INFINITY;
  bool bad = false;
  s.each([&](int i, float x) {
    top = fmaxf(top, x);
    least = fminf(least, x);
    bad |= x != x && i < a.V;
  });
  top = wave_max(top);
  least = wave_min(least);
  bad = __any(bad);
  if (s.lane == 0) sh.top[s.wave] = bad ? NAN : top, sh.least[s.wave] = least;
  if (threadIdx.x == 0) sh.first = 0x7fffffffu;
  __syncthreads();
  bool nan = false;
#pragma unroll
  for (int q = 0; q < S::NT / 64; ++q) {
    const float its = sh.top[q];
    nan |= its != its;
    top = fmaxf(top, its), least = fminf(least, sh.least[q]);
  }
  s.top = top;
  s.least = least;
  const float t = a.temperature ? a.temperature[r] : a.t0;
  if (nan || !(t > 0.f)) {
    // the first NaN, which is above all as in torch's argmax, or the first of the largest
    uint32_t at = 0x7fffffffu;
    s.each([&](int i, float x) {
      if ((nan ? x != x : x == top) && i < a.V) at = min(at, (uint32_t)i);
    });
    if (at != 0x7fffffffu) atomicMin(&sh.first, at);
    __syncthreads();
    return (int)sh.first;
  } else {
    s.c = 1.4426950408889634 / (double)t;
    // every logit above the last bin, but what lies 31 temperatures below the largest
    s.width = (float)(S::B - 1) / fminf((top - least) * 1.001f, 31.f * t);
    if (!(s.width > 0.f && s.width < 3e38f)) s.width = 0.f;
    const typename S::Kept kept(s.border(a.top_k ? a.top_k[r] : a.k0, a.top_p ? a.top_p[r] : a.p0));
    const float m = a.min_p ? a.min_p[r] : a.m0, u = a.uniform[r];
    const double least_x = m >= 1.f ? (double)top : m > 0.f ? (double)top + (double)t * log((double)m) : -INFINITY;
    return s.find([&](int i, float x) { return kept(i, x) && !((double)x < least_x) ? s.weight(x) : (uint64_t)0; },
                    [&](uint64_t sum) {
                      const double f = u > 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
                      return (uint64_t)(f * (double)sum);
                    });
  }
}

template <typename S>
__device__ __forceinline__ void sample_power_table(S& s) {
  for (int j = threadIdx.x; j < 256; j += S::NT) s.sh->power[j] = exp2(j / 256.0);
}

template <typename T, int NW>
__global__ void __launch_bounds__(64 * NW) sample_tokens_kernel(SampleArgs a) {
  using S = Sampler<T, NW>;
  __shared__ typename S::Shared shared;
  S s;
  s.sh = &shared;
  s.start(a, blockIdx.x, 0, (a.V + kSampleChunk - 1) / kSampleChunk);
  sample_power_table(s);
  const int answer = sample_row(s, a, blockIdx.x);
  if (threadIdx.x == 0) a.ids[blockIdx.x] = answer;
}

// ------------------------------------------------------------------------------------------------ few long rows
// Rows too few to fill the card are cut into parts of 8 chunks and more, a workgroup each, and the passes above become launches: the
// parts' largest logits; their bins; where a top-k is asked for, the tokens of its border's bin; the chunks' weights above the
// last border's bin, and that bin's tokens; and a workgroup a row that orders these, adds what is kept of them to the chunks' sums and finds
// the token.  What a launch needs of the ones before (the largest logit, the bins' sums, the borders' bins) each workgroup joins for itself, in
// the same way: nothing is added up in memory, and nothing is waited for.  A row with a NaN, without a temperature, or with more tokens in a border's
// bin than the list holds is answered by the last launch alone, as a single workgroup does.
constexpr int kWideParts = 32, kWideBins = 1024, kWideList = 1024;

struct WideRow {
  float *top, *least;         // of each part; a NaN: one is there
  unsigned long long* ends;   // where the filters end: Wide's members behind borders(), and whether it found them
  unsigned long long* chunk;  // the kept weights of each chunk, but the border's bin
  unsigned long long* mass;   // the bins of each part
  uint32_t* count;
  uint32_t* n;                      // two lists of each part: the tokens of a border's bin
  unsigned long long *key, *weight;
  __host__ __device__ static int64_t bytes(int parts, int chunks) {
    return 64 + 2 * 8 * (int64_t)kWideParts + 8 * (int64_t)chunks + parts * (12 * (int64_t)kWideBins + 2 * 16 * (int64_t)kWideList);
  }
  __device__ __forceinline__ WideRow(const SampleArgs& a, int64_t r, int chunks) {
    uint8_t* p = a.held + r * bytes(a.parts, chunks);
    ends = (unsigned long long*)p, p += 64;
    chunk = (unsigned long long*)p, p += 8 * (int64_t)chunks;
    mass = (unsigned long long*)p, p += 8 * (int64_t)kWideBins * a.parts;
    key = (unsigned long long*)p, p += 16 * (int64_t)kWideList * a.parts;
    weight = (unsigned long long*)p, p += 16 * (int64_t)kWideList * a.parts;
    count = (uint32_t*)p, p += 4 * (int64_t)kWideBins * a.parts;
    top = (float*)p, least = top + kWideParts, n = (uint32_t*)(least + kWideParts);  // (n: two for each part)
  }
};

// Parts of a row's chunks, or 0: a workgroup a row.  us, a workgroup a row / shared, fp32 without a filter, with top-p, top-k, both:
//   16,001 logits,  1 row  12.2 / 12.5   20.7 / 21.3   16.2 / 23.1   23.5 / 27.3
//   30,000          1      18.1 / 13.0   31.7 / 22.8   21.7 / 25.1   33.2 / 29.3
//   50,304          1      27.0 / 13.1   43.1 / 22.9   30.7 / 26.9   48.1 / 31.7
//   50,304         32      28.0 / 15.6   48.4 / 34.0   31.4 / 33.1   49.5 / 44.0
//   2^20            1       396 / 30      648 / 59      397 / 49      679 / 62
//   2^20           16       398 / 49      661 / 93      398 / 77      681 / 98
static int wide_parts(int64_t rows, int64_t V, int dtype) {
  const int chunks = (int)((V + kSampleChunk - 1) / kSampleChunk);
  if ((dtype_size(dtype) == 2 && V < 65536) || chunks < 64) return 0;
  const int parts = std::min((chunks + 7) / 8, kWideParts);
  return rows * parts <= 2 * device_cu_count() ? parts : 0;
}

template <typename T>
struct Wide : Sampler<T, 8, kWideBins, kWideList> {
  using S = Sampler<T, 8, kWideBins, kWideList>;
  using S::NT, S::sh, S::lane, S::wave, S::top, S::least, S::c, S::width, S::V;
  static constexpr int B = kWideBins;
  WideRow w;
  int parts, part, chunks;
  float t;
  double least_x;           // a kept token's least value
  int border = B;           // the last border's bin; B: none
  int listed = -1;          // top-k's border's bin, where list 0 has its tokens
  uint64_t keep = 0;        // the last token that top-k keeps
  uint64_t above = 0, target = 0;  // top-p's border: the weight above its bin, and where it ends

  __device__ __forceinline__ Wide(const SampleArgs& a, int64_t r, int first_part, int last_part, typename S::Shared* shared)
      : w(a, r, (a.V + kSampleChunk - 1) / kSampleChunk) {
    sh = shared;
    parts = a.parts, part = first_part, chunks = (a.V + kSampleChunk - 1) / kSampleChunk;
    const int per = (chunks + parts - 1) / parts;
    S::start(a, r, min(first_part * per, chunks), min(last_part * per, chunks));
    t = a.temperature ? a.temperature[r] : a.t0;
  }

  // The row's largest and smallest logit from its parts'; whether the launches share this row
  __device__ __forceinline__ bool join(const SampleArgs& a, int64_t r) {
    const float x = lane < parts ? w.top[lane] : -INFINITY, y = lane < parts ? w.least[lane] : INFINITY;
    const bool nan = __any(x != x);
    top = wave_max(x);
    least = wave_min(y);
    if (nan || !(t > 0.f)) return false;
    sample_power_table(*this);
    c = 1.4426950408889634 / (double)t;
    width = (float)(B - 1) / fminf((top - least) * 1.001f, 31.f * t);
    if (!(width > 0.f && width < 3e38f)) width = 0.f;
    const float m = a.min_p ? a.min_p[r] : a.m0;
    least_x = m >= 1.f ? (double)top : m > 0.f ? (double)top + (double)t * log((double)m) : -INFINITY;
    __syncthreads();
    return true;
  }
  __device__ __forceinline__ bool by_count(const SampleArgs& a, int64_t r, int& k) const {
    k = a.top_k ? a.top_k[r] : a.k0;
    return k > 0 && k < V;
  }
  __device__ __forceinline__ bool by_mass(const SampleArgs& a, int64_t r, float& p) const {
    p = a.top_p ? a.top_p[r] : a.p0;
    return p < 1.f;
  }

  // The sum over the parts of each bin's count or mass, in LDS; eight parts' loads at once
  template <typename A>
  __device__ __forceinline__ void join_bins(const A* from, A* to) {
    for (int b = threadIdx.x; b < B; b += NT) {
      A sum = 0;
#pragma unroll 1
      for (int q = 0; q < parts; q += 8) {
        A v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = q + i < parts ? from[(q + i) * B + b] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
      }
      to[b] = sum;
    }
  }
  // A list's tokens, joined in LDS
  __device__ __forceinline__ int join_list(int which) {
    const uint32_t its = lane < parts ? min(w.n[2 * lane + which], (uint32_t)kWideList) : 0, upto = wave_scan32(its);
    const int n = min((int)lane32(upto, 63), kWideList);  // (a row with more is not shared)
#pragma unroll 1
    for (int q = wave; q < parts; q += NT / 64) {
      const int own = (int)lane32(its, q), at = (int)lane32(upto, q) - own;
      const int64_t from = (int64_t)(2 * q + which) * kWideList;
      for (int j = lane; j < own && at + j < kWideList; j += 64) sh->key[at + j] = w.key[from + j], sh->weight[at + j] = w.weight[from + j];
    }
    __syncthreads();
    return n;
  }
  // Top-k's border's bin, B: none; false where its bin holds too many
  __device__ __forceinline__ bool count_border(int k, int& b) {
    uint64_t before, held;
    b = S::template find_bin<S::BPER>(sh->count, 0, (uint64_t)k, before, held);
    above = before;
    if (b == B - 1) b = B;
    return b == B || held <= kWideList;
  }
  // Where the row's filters end; false where a bin holds too many tokens for the list
  __device__ __forceinline__ bool borders(const SampleArgs& a, int64_t r) {
    int k;
    float p;
    const bool count = by_count(a, r, k), mass = by_mass(a, r, p);
    if (!count && !mass) return true;
    if (count) join_bins(w.count, sh->count);
    if (mass) join_bins(w.mass, sh->mass);
    __syncthreads();
    uint64_t total = 0, held;
    if (count) {
      int b;
      if (!count_border(k, b)) return false;
      if (b < B) {
        listed = border = b;
        const int n = join_list(0);
        const uint64_t before = above;
        keep = S::cut(n, [&](uint32_t rank, uint64_t) { return before + rank < (uint64_t)k; }, total);
      }
    }
    if (!mass) return true;
    uint64_t mine = 0;
#pragma unroll
    for (int j = 0; j < S::BPER; ++j)
      if (listed < 0 || (int)(S::BPER * threadIdx.x + j) < listed) mine += sh->mass[S::BPER * threadIdx.x + j];
    total += S::block_sum(mine);
    const double want = (double)p * (double)total;
    target = min(max((uint64_t)(want > 0.0 ? ceil(want) : 1.0), (uint64_t)1), total);
    border = S::template find_bin<S::BPER>(sh->mass, 0, target, above, held);
    return lane32(wave_scan32(lane < parts ? w.count[lane * B + border] : 0), 63) <= (uint32_t)kWideList;
  }
  __device__ __forceinline__ void store_ends(bool found) const {
    w.ends[0] = found, w.ends[1] = (unsigned)border, w.ends[2] = (unsigned)listed, w.ends[3] = keep, w.ends[4] = above, w.ends[5] = target;
  }
  __device__ __forceinline__ bool load_ends() {
    border = (int)w.ends[1], listed = (int)(unsigned)w.ends[2], keep = w.ends[3], above = w.ends[4], target = w.ends[5];
    return w.ends[0] != 0;
  }
  // This part's tokens of bin b into list `which`, and done(chunk) behind each chunk's f(value, bin)
  template <typename F, typename D>
  __device__ __forceinline__ void list_tokens(int b, int which, F f, D done) {
    if (threadIdx.x == 0) sh->n = 0;
    __syncthreads();
    const int64_t from = (int64_t)(2 * part + which) * kWideList;
    S::each(
        [&](int i, float x) {
          const int its = S::bin(x);
          f(x, its);
          if (its == b && x == x) {
            const uint32_t at = atomicAdd(&sh->n, 1u);
            if (at < (uint32_t)kWideList) w.key[from + at] = sample_order(SampleKey<T>::of_value(x), i), w.weight[from + at] = S::weight(x);
          }
        },
        done);
    __syncthreads();
    if (threadIdx.x == 0) w.n[2 * part + which] = sh->n;
  }
};

template <typename T>
__global__ void __launch_bounds__(512) wide_top_kernel(SampleArgs a) {
  __shared__ typename Wide<T>::Shared shared;
  Wide<T> s(a, blockIdx.y, blockIdx.x, blockIdx.x + 1, &shared);
  float top = -INFINITY, least = INFINITY;
  bool bad = false;
  s.each([&](int i, float x) {
    top = fmaxf(top, x);
    least = fminf(least, x);
    bad |= x != x && i < a.V;
  });
  top = wave_max(top);
  least = wave_min(least);
  if (__any(bad)) top = NAN;
  if (s.lane == 0) shared.top[s.wave] = top, shared.least[s.wave] = least;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int q = 1; q < 8; ++q) {
      const float its = shared.top[q];
      top = its != its || top != top ? NAN : fmaxf(top, its);
      least = fminf(least, shared.least[q]);
    }
    s.w.top[s.part] = top;
    s.w.least[s.part] = least;
  }
}

template <typename T>
__global__ void __launch_bounds__(512) wide_bins_kernel(SampleArgs a) {
  using W = Wide<T>;
  __shared__ typename W::Shared shared;
  W s(a, blockIdx.y, blockIdx.x, blockIdx.x + 1, &shared);
  int k;
  float p;
  const bool count = s.by_count(a, blockIdx.y, k), mass = s.by_mass(a, blockIdx.y, p);
  if (!(count || mass) || !s.join(a, blockIdx.y)) return;
  for (int b = threadIdx.x; b < W::B; b += W::NT) shared.mass[b] = 0, shared.count[b] = 0;
  __syncthreads();
  s.each([&](int, float x) {  // (a missing one is counted in the last bin, where it changes nothing)
    const int b = s.bin(x);
    atomicAdd(&shared.count[b], 1u);
    if (mass) atomicAdd(&shared.mass[b], (unsigned long long)s.weight(x));
  });
  __syncthreads();
  for (int b = threadIdx.x; b < W::B; b += W::NT) {
    s.w.count[s.part * W::B + b] = shared.count[b];
    if (mass) s.w.mass[s.part * W::B + b] = shared.mass[b];
  }
}

// Top-k's border's tokens
template <typename T>
__global__ void __launch_bounds__(512) wide_list_kernel(SampleArgs a) {
  using W = Wide<T>;
  __shared__ typename W::Shared shared;
  W s(a, blockIdx.y, blockIdx.x, blockIdx.x + 1, &shared);
  int k, b;
  if (!s.by_count(a, blockIdx.y, k) || !s.join(a, blockIdx.y)) return;
  s.join_bins(s.w.count, shared.count);
  __syncthreads();
  if (!s.count_border(k, b) || b == W::B) return;
  s.list_tokens(b, 0, [](float, int) {}, [](int) {});
}

// The chunks' weights above the last border's bin; top-p's border's tokens
template <typename T>
__global__ void __launch_bounds__(512) wide_sums_kernel(SampleArgs a) {
  using W = Wide<T>;
  __shared__ typename W::Shared shared;
  W s(a, blockIdx.y, blockIdx.x, blockIdx.x + 1, &shared);
  if (!s.join(a, blockIdx.y)) return;
  const bool found = s.borders(a, blockIdx.y);
  if (s.part == 0 && threadIdx.x == 0) s.store_ends(found);
  if (!found) return;
  uint64_t own = 0;
  s.list_tokens(s.border == s.listed ? -1 : s.border, 1,
                [&](float x, int b) { own += b < s.border && !((double)x < s.least_x) ? s.weight(x) : 0; },
                [&](int q) {
                  own = wave_sum64(own);
                  if (s.lane == 0) s.w.chunk[q] = own;
                  own = 0;
                });
}

template <typename T>
__global__ void __launch_bounds__(512) wide_pick_kernel(SampleArgs a) {
  using W = Wide<T>;
  __shared__ typename W::Shared shared;
  const int64_t r = blockIdx.x;
  W s(a, r, 0, a.parts, &shared);
  int answer;
  if (!s.join(a, r) || !s.load_ends()) {
    __syncthreads();
    sample_power_table(s);
    answer = sample_row((typename W::S&)s, a, r);
  } else {
    uint64_t last = s.keep;
    int n = 0;
    if (s.border < W::B) {
      n = s.join_list(s.border == s.listed ? 0 : 1);
      uint64_t sum;
      if (s.target) last = max(last, s.cut(n, [&](uint32_t, uint64_t before) { return s.above + before < s.target; }, sum));
    }
    for (int q = threadIdx.x; q < s.chunks; q += W::NT) shared.mass[q] = s.w.chunk[q];
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += W::NT) {
      const uint64_t k = shared.key[j];
      if (k >= last && !((double)SampleKey<T>::value((uint32_t)(k >> 32)) < s.least_x))
        atomicAdd(&shared.mass[(int)~(uint32_t)k / kSampleChunk], (unsigned long long)shared.weight[j]);
    }
    const typename W::Kept kept(last);
    const float u = a.uniform[r];
    answer = s.find_in_chunks([&](int i, float x) { return kept(i, x) && !((double)x < s.least_x) ? s.weight(x) : (uint64_t)0; },
                              [&](uint64_t sum) {
                                const double f = u > 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
                                return (uint64_t)(f * (double)sum);
                              });
  }
  if (threadIdx.x == 0) a.ids[r] = answer;
}

// ------------------------------------------------------------------------------------------------ 16-bit logits
// Rows of up to 65,535 16-bit logits hold at most 65,536 different values: one pass over the row counts every value in LDS (two
// 16-bit counters a word), and the filters are decided on values and counts alone, a weight for each value that occurs.  In
// falling order the words are 32 strips of 1,024, a word a thread; a strip's wave that holds any leaves its count and
// weight in a table of 512 entries, and each wave finds a border there, then in the entry's words.  A last pass over the row adds
// up the kept weights, and counts the tokens of the border's value, of which the first so many are kept; each lane leaves both
// for each of its chunks in LDS, where the wave in whose part the answer lies finds it.
//
// 32 rows of 50,304 with mixed filters take 23 to 26 us (the row with the most kept tokens), 2,048 rows 157, 1.3 TB/s: eight rows a CU one after
// the other, a third of it the count (LDS atomics, 11 cycles a wave's), a fifth the kept weights.
//
// Keys here are the 16 bits in the values' order as they are: NaNs lie at both ends, and -0, 0x7fff, is counted as +0, 0x8000.
constexpr int kCountedThreads = 1024, kCountedChunks = 8;  // 512 logits a chunk and wave

template <typename T>
__device__ __forceinline__ uint32_t ordered2(uint32_t x) {  // of two logits
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  return x ^ (__builtin_bit_cast(uint32_t, __builtin_bit_cast(s16x2, x) >> 15) | 0x80008000u);
}
template <typename T>
__device__ __forceinline__ float ordered_value(uint32_t key) {
  return to_f32(__builtin_bit_cast(T, (uint16_t)(key & 0x8000u ? key ^ 0x8000u : ~key)));
}

template <typename T>
struct Counted {
  static constexpr uint32_t kInf = __is_same(T, bf16) ? 0xff80u : 0xfc00u, kNegInf = 0xffffu - kInf;
  // the weights' tables: mantissa bits and the upper ones of them, exponents a sign
  static constexpr int kMan = __is_same(T, bf16) ? 7 : 10, kBias = __is_same(T, bf16) ? 127 : 15, kHigh = (kMan + 1) / 2,
                       kLow = kMan - kHigh, kExps = __is_same(T, bf16) ? 32 : 30;
  static constexpr int kHighs = (kExps << kHigh) + 1, kLows = (kExps + 1) << kLow;  // a sign's, and behind them a weight of 0
  struct Shared {
    union {
      uint32_t table[32768];
      struct {
        unsigned long long own[kCountedChunks][kCountedThreads];  // a lane's weight in a chunk
        uint32_t same[kCountedChunks][kCountedThreads];           // and its tokens of the border's value
        double high[2 * kHighs], low[2 * kLows];
      };
    };
    unsigned long long mass[512];
    uint32_t count[512];
    double power[256];
    unsigned long long part[16], n, one;
    uint32_t ties[16];
    unsigned top, first, at, low_key, least, nan;
  };
  static_assert(sizeof(((Shared*)0)->own) + sizeof(((Shared*)0)->same) + sizeof(((Shared*)0)->high) + sizeof(((Shared*)0)->low) <=
                    sizeof(((Shared*)0)->table), "they take the counts' place");
  Shared* sh;
  const uint16_t* row;
  int V, lane, wave, first, chunks;  // the wave's part of the row: its first chunk and their number
  uint32_t top, strips;              // strips of which the wave's words hold any
  double xmax, c;
  int least_exp;                     // the first exponent that the weights' tables hold

  __device__ __forceinline__ int index(int q) const { return (first + q) * kSampleChunk + 8 * lane; }
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    const uint64_t w = sample_weight((double)ordered_value<T>(k), xmax, c, sh->power);
    return k == top ? kSampleOne : w;
  }
  // The logits of chunk q; what lies behind the row's end reads as 0xffff, key 0
  __device__ __forceinline__ u32x4 load(int q) const {
    const int i = index(q);
    if ((first + q + 1) * kSampleChunk <= V) return *(const u32x4_at2*)(row + i);
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      v[e >> 1] = (i + e < V ? row[i + e] : 0xffffu) | (i + e + 1 < V ? row[i + e + 1] : 0xffffu) << 16;
    return v;
  }
  // f(chunk, its logits, two a word), loads two chunks ahead (a and b: the first two)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    u32x4 a = {}, b = {};
    if (chunks > 0) a = load(0);
    if (chunks > 1) b = load(1);
    each(a, b, f);
  }
  template <typename F>
  __device__ __forceinline__ void each(u32x4 a, u32x4 b, F f) const {
#pragma unroll 1
    for (int q = 0; q < chunks; ++q) {
      const u32x4 now = a;
      a = b;
      if (q + 2 < chunks) b = load(q + 2);
      f(q, now);
    }
  }
  static __device__ __forceinline__ uint32_t half(uint32_t pair, int e) { return e & 1 ? pair >> 16 : pair & 0xffffu; }

  __device__ __forceinline__ void count_values(const u32x4& a, const u32x4& b) {
    each(a, b, [&](int, const u32x4& raw) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t k = ordered2<T>(raw[e]);
        uint8_t* t = (uint8_t*)sh->table;
        atomicAdd((uint32_t*)(t + ((k << 1) & 0x1fffcu)), (k & 1) * 65535u + 1);
        atomicAdd((uint32_t*)(t + ((k >> 15) & 0x1fffcu)), ((k >> 16) & 1) * 65535u + 1);
      }
    });
  }

  // The first index whose key is in [lo, hi] or [lo2, hi2]
  __device__ __forceinline__ int first_of(uint32_t lo, uint32_t hi, uint32_t lo2, uint32_t hi2) {
    int at = 0x7fffffff;
    each([&](int q, const u32x4& raw) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t k = half(ordered2<T>(raw[e >> 1]), e);
        const int i = index(q) + e;
        if (((k >= lo && k <= hi) || (k >= lo2 && k <= hi2)) && i < V) at = min(at, i);
      }
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, 64));
    if (lane == 0) atomicMin(&sh->first, (unsigned)at);
    __syncthreads();
    return (int)sh->first;
  }

  // Counts and weights of the entries (cleared before): strip i, wave w of the words in falling order
  __device__ __forceinline__ void tabulate(bool weights) {
    for (uint32_t left = strips; left; left &= left - 1) {
      const int i = __builtin_ctz(left), at = 1024 * i + threadIdx.x;
      const uint32_t word = sh->table[32767 - at], k = 65535u - 2 * at;
      if (!__any(word != 0)) continue;
      const uint32_t n = wave_scan32((word >> 16) + (word & 0xffffu));
      if (lane == 63) sh->count[16 * i + wave] = n;
      if (weights) {
        const uint64_t m = wave_scan64((word >> 16) * weight(k) + (word & 0xffffu) * weight(k - 1));
        if (lane == 63) sh->mass[16 * i + wave] = m;
      }
    }
    __syncthreads();
  }

  // The value at which the tokens in order first hold `target` (>= 1, at most the whole sum): its key, the sum before it and how
  // many hold it
  template <bool MASS, typename A>
  __device__ __forceinline__ uint32_t border(A target, A& above, uint32_t& number) const {
    A v[8], mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine += v[j] = MASS ? (A)sh->mass[8 * lane + j] : (A)sh->count[8 * lane + j];
    A at = wave_scan(mine) - mine;
    int entry = -1;
    const bool here = at < target && at + mine >= target;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (here && entry < 0) {
        if (at + v[j] >= target) entry = 8 * lane + j;
        else at += v[j];
      }
    }
    const int l = __builtin_ctzll(__ballot(here));
    entry = (int)lane32((uint32_t)entry, l);
    at = lane_of(at, l);
    const int pos = 1024 * (entry >> 4) + 64 * (entry & 15) + lane;
    const uint32_t word = sh->table[32767 - pos], k = 65535u - 2 * pos;
    A hi = word >> 16, lo = word & 0xffffu;
    if constexpr (MASS) hi *= weight(k), lo *= weight(k - 1);
    at += wave_scan(hi + lo) - hi - lo;
    const bool this_one = at < target && at + hi + lo >= target, low = at + hi < target;
    const int l2 = __builtin_ctzll(__ballot(this_one));
    above = lane_of(low ? at + hi : at, l2);
    number = lane32(low ? word & 0xffffu : word >> 16, l2);
    return lane32(low ? k - 1 : k, l2);
  }

  // The weight of every value above key k
  __device__ __forceinline__ uint64_t weight_above(uint32_t k) const {
    const int pos = (int)(65535u - k) >> 1, entry = 16 * (pos >> 10) + ((pos >> 6) & 15);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += 8 * lane + j < entry ? (uint64_t)sh->mass[8 * lane + j] : 0;
    const int p = 1024 * (entry >> 4) + 64 * (entry & 15) + lane;
    const uint32_t word = sh->table[32767 - p], kp = 65535u - 2 * p;
    if (kp > k) sum += (word >> 16) * weight(kp);
    if (kp - 1 > k) sum += (word & 0xffffu) * weight(kp - 1);
    return wave_sum64(sum);
  }

  // The least value with its share m of the largest weight, as a key; every value is above key 0
  __device__ __forceinline__ uint32_t least_key(float m, float t) const {
    if (!(m > 0.f)) return 1;
    const double x = m >= 1.f ? xmax : xmax + (double)t * log((double)m);
    uint32_t least = ordered2<T>(__builtin_bit_cast(uint16_t, from_f32<T>((float)x))) & 0xffffu;
    if (least == 0x7fffu) least = 0x8000u;
    // (rounded twice and either way: at most a value off; a NaN, of infinities, keeps all)
    if (x != x) return 1;
    while (least > kNegInf && (double)ordered_value<T>(least - 1) >= x) --least;
    while (least < kInf && (double)ordered_value<T>(least) < x) ++least;
    return least == 0x8000u ? 0x7fffu : least;
  }

  // What is kept (one wave finds it): every value above `at`, and the first n tokens of those with keys from `low` to `at` (none where
  // low > at)
  __device__ __forceinline__ void filter(int k, float p) {
    const bool by_count = k > 0 && k < V, by_mass = p < 1.f;
    uint32_t at = 0, low = 1;
    uint64_t n = 0;
    uint32_t number;
    if (by_count || by_mass) {
      bool cut = false;
      if (by_count) {
        uint32_t above;
        at = border<false>((uint32_t)k, above, number);
        n = (uint32_t)k - above;
        cut = n < number;
      }
      if (by_mass) {
        const uint64_t total = weight_above(at) + (by_count ? n * weight(at) : 0);
        const double want = (double)p * (double)total;
        const uint64_t target = min(max((uint64_t)(want > 0.0 ? ceil(want) : 1.0), (uint64_t)1), total);
        uint64_t above;
        const uint32_t pk = border<true>(target, above, number);
        // the least number of them that holds what is missing
        const uint64_t w = weight(pk), missing = target - above;
        uint64_t take = (uint64_t)((double)missing / (double)w);
        while (take * w < missing) ++take;
        while (take > 1 && (take - 1) * w >= missing) --take;
        if (pk != at || take < n) {
          cut = (pk == at && cut) || take < number;
          n = take;
        }
        at = pk;
      }
      low = at == 0x8000u ? 0x7fffu : at;
      if (!cut) at = low - 1, low = at + 1;
    }
    if (lane == 0) {
      sh->at = at;
      sh->low_key = low;
      sh->n = n;
      sh->one = low <= at ? weight(at) : 0;
    }
  }

  // Weights by tables, for rows that keep many tokens.  x = s (2^E + f) for each sign and exponent E, its fraction f = f1 + f2 by its
  // upper and lower bits: 2^43 exp((s (2^E + f1) - max) / t) times exp(s f2 / t), 24 (fp16: 64) values a binade, for the binades up
  // to the largest magnitude that has a weight.  Returns whether they serve (else a factor might leave fp64's range)
  __device__ __forceinline__ bool prepare(float t) {
    const float most = fabsf((float)xmax) + 31.f * t;
    const uint32_t bits = __builtin_bit_cast(uint16_t, from_f32<T>(most * 1.01f)) & 0x7fffu;
    const int hi = min((int)(bits >> kMan), (1 << (15 - kMan)) - 2);  // (the last exponent is that of infinities)
    least_exp = max(hi - kExps + 1, 0);
    const double ulp = __builtin_amdgcn_ldexp(1.0, max(hi, 1) - kBias - kMan);
    if (!(ulp * c * (1 << kLow) < 500.0) || !(fabs(xmax) < 1e30)) return false;
    for (int i = threadIdx.x; i < 2 * (kHighs + kLows); i += kCountedThreads) {
      const bool upper = i < 2 * kHighs;
      const int size = upper ? kHighs : kLows, shift = upper ? kHigh : kLow;
      int j = upper ? i : i - 2 * kHighs;
      const bool negative = j >= size;
      if (negative) j -= size;
      const int E = (j >> shift) + least_exp, f = (j & ((1 << shift) - 1)) << (upper ? kLow : 0);
      double x = __builtin_amdgcn_ldexp((double)(f + (upper && E ? 1 << kMan : 0)), max(E, 1) - kBias - kMan);
      if (negative) x = -x;
      const double y = upper ? fma(x - xmax, c, 43.0) : x * c;
      double w = sample_power(fmin(fmax(y, -1000.0), 1000.0), sh->power);
      if (j >> shift == kExps) w = 0.0;
      (upper ? sh->high : sh->low)[i - (upper ? 0 : 2 * kHighs)] = w;
    }
    return true;
  }
  // The sum of the weights of chunk elements kept by `keep`, one multiplication and addition each: 2^52 + (a whole number) rounds
  // every addition to a whole number.  Magnitudes above the tables' belong to negative logits without a weight
  __device__ __forceinline__ double table_add(double sum, uint32_t raw, bool keep) const {
    const uint32_t mag = raw & 0x7fffu, sign = raw >> 15;
    const uint32_t at = min((mag >> kLow) - ((uint32_t)least_exp << kHigh), (uint32_t)(kExps << kHigh));
    const uint32_t hi = keep ? at + sign * kHighs : (uint32_t)(kExps << kHigh);
    const uint32_t lo = ((at >> kHigh) << kLow) + (mag & ((1 << kLow) - 1)) + sign * kLows;
    return fma(sh->high[hi], sh->low[lo], sum);
  }
  // The kept weight of eight logits, and up to the e-th
  __device__ __forceinline__ uint64_t table_weight8(const u32x4& raw, uint32_t at) const {
    double sum = 0x1p52;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = table_add(sum, half(raw[e >> 1], e), half(ordered2<T>(raw[e >> 1]), e) > at);
    return __builtin_bit_cast(uint64_t, sum) & 0xfffffffffffffull;
  }
  // Whether a chunk's weights are best looked up: three steps and more of its eight meet a kept token, and the tables hold the
  // magnitudes of all its logits (none lies below them)
  __device__ __forceinline__ bool held(const u32x4& raw, uint32_t at) const {
    uint32_t least = 0x7fffu;
    int steps = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      least = min(least, half(raw[e >> 1], e) & 0x7fffu);
      steps += __any(half(ordered2<T>(raw[e >> 1]), e) > at) != 0;
    }
    return steps >= 3 && !__any((int)(least >> kMan) < least_exp);
  }

  // The kept weights, and the border's tokens, of the wave's part
  template <bool TABLES>
  __device__ __forceinline__ void add_up(uint32_t at, uint32_t low, uint64_t& sum, uint32_t& number) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const bool ties = low <= at;
    const uint32_t least = ties ? low : at + 1;
    each([&](int q, const u32x4& raw) {
      uint64_t own = 0;
      uint32_t same = 0;
      u16x2 most = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, ordered2<T>(raw[e])));
      if (!__any(max((uint32_t)most[0], (uint32_t)most[1]) >= least)) {  // nothing kept
        sh->own[q][threadIdx.x] = 0;
        sh->same[q][threadIdx.x] = 0;
        return;
      }
      if (TABLES && held(raw, at)) {
        own = table_weight8(raw, at);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = half(ordered2<T>(raw[e >> 1]), e);
          if (__any(key > at)) own += key > at ? weight(key) : 0;
        }
      }
      if (ties) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = half(ordered2<T>(raw[e >> 1]), e);
          same += key - low <= at - low;
        }
      }
      sh->own[q][threadIdx.x] = own;
      sh->same[q][threadIdx.x] = same;
      sum += own;
      number += same;
    });
  }
};

template <typename T>
__global__ void __launch_bounds__(kCountedThreads) sample_counted_kernel(SampleArgs a) {
  using S = Counted<T>;
  __shared__ typename S::Shared shared;
  S s;
  s.sh = &shared;
  s.V = a.V;
  s.lane = threadIdx.x & 63;
  s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunks = (a.V + kSampleChunk - 1) / kSampleChunk, each = (chunks + 15) / 16;
  s.first = min(s.wave * each, chunks);
  s.chunks = min(each, chunks - s.first);
  if (threadIdx.x < 256) shared.power[threadIdx.x] = exp2(threadIdx.x / 256.0);
  const int64_t r = blockIdx.x;
  s.row = (const uint16_t*)a.logits + r * a.ld;
  u32x4 first = {}, second = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) ((u32x4*)shared.table)[1024 * i + threadIdx.x] = u32x4{};
  if (threadIdx.x < 512) shared.count[threadIdx.x] = 0, shared.mass[threadIdx.x] = 0;
  if (threadIdx.x == 0) shared.top = 0xffffffffu, shared.first = 0x7fffffffu, shared.nan = 0;
  __syncthreads();
  if (s.chunks > 0) first = s.load(0);
  if (s.chunks > 1) second = s.load(1);
  s.count_values(first, second);
  __syncthreads();
  // ---- the largest value; NaNs lie in the first and the last strip (what lies behind the row's end is counted at key 0)
  bool bad = false;
  const uint32_t behind = (uint32_t)(chunks * kSampleChunk - a.V);
  // four strips at a time, four words a lane: the wave's 64 of each
  uint32_t strips = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = 1024 * (4 * i + (s.lane >> 4)) + 64 * s.wave + 4 * (s.lane & 15);
    u32x4 words = *(const u32x4*)&shared.table[32764 - at];
    if (i == 7 && at == 32764) words[0] -= behind;
    strips |= ((words[0] | words[1] | words[2] | words[3]) != 0 ? 1u : 0u) << (4 * i);
  }
  s.strips = wave_or32(strips << (s.lane >> 4));
  constexpr int nans = (0x10000 - S::kInf) / 2;  // words of either end that hold NaNs
  if (s.wave < nans / 64) {
    const uint32_t word = shared.table[32767 - threadIdx.x], k = 65535u - 2 * threadIdx.x;
    bad = (word >> 16 && k > S::kInf) || (word & 0xffffu && k - 1 > S::kInf);
  }
  if (s.wave >= 16 - nans / 64) {
    const uint32_t word = shared.table[1023 - threadIdx.x] - (threadIdx.x == 1023 ? behind : 0), k = 2047u - 2 * threadIdx.x;
    bad |= (word >> 16 && k < S::kNegInf) || (word & 0xffffu && k - 1 < S::kNegInf);
  }
  if (s.strips) {
    const int at = 1024 * __builtin_ctz(s.strips) + threadIdx.x;
    const uint32_t word = shared.table[32767 - at];
    const int l = __builtin_ctzll(__ballot(word != 0));
    if (s.lane == l) atomicMin(&shared.top, 2u * at + (word >> 16 ? 0 : 1));
  }
  if (bad) shared.nan = 1;
  __syncthreads();
  const bool nan = shared.nan != 0;
  s.top = 65535u - shared.top;
  if (threadIdx.x == 0) {
    shared.table[0] &= 0xffff0000u;
    const uint32_t zeros = shared.table[0x3fff] >> 16;  // -0
    shared.table[0x3fff] &= 0xffffu;
    shared.table[0x4000] += zeros;
  }
  s.strips |= 1u << 15;  // (where +0 lies)
  if (s.top == 0x7fffu) s.top = 0x8000u;
  __syncthreads();
  const float t = a.temperature ? a.temperature[r] : a.t0;
  if (nan) {
    const int i = s.first_of(S::kInf + 1, 0xffffu, 0, S::kNegInf - 1);
    if (threadIdx.x == 0) a.ids[r] = i;
  } else if (!(t > 0.f)) {
    const int i = s.first_of(s.top == 0x8000u ? 0x7fffu : s.top, s.top, 1, 0);
    if (threadIdx.x == 0) a.ids[r] = i;
  } else {
    s.xmax = (double)ordered_value<T>(s.top);
    s.c = 1.4426950408889634 / (double)t;
    const int k = a.top_k ? a.top_k[r] : a.k0;
    const float p = a.top_p ? a.top_p[r] : a.p0, m = a.min_p ? a.min_p[r] : a.m0, u = a.uniform[r];
    if ((k > 0 && k < a.V) || p < 1.f) s.tabulate(p < 1.f);
    if (s.wave == 0) s.filter(k, p);
    if (s.wave == 1 && s.lane == 0) shared.least = s.least_key(m, t);
    __syncthreads();  // the counts are read
    uint32_t at = shared.at, low = shared.low_key;
    if (shared.least > at + (low <= at ? 0 : 1)) at = shared.least - 1, low = at + 1;
    const uint64_t n = shared.n, one = low <= at ? shared.one : 0;
    // tables pay where most waves meet a kept token at most of their steps
    const bool tables = (k <= 0 || k > 512) && s.prepare(t);
    __syncthreads();
    uint64_t sum = 0;
    uint32_t number = 0;
    if (tables) s.template add_up<true>(at, low, sum, number);
    else s.template add_up<false>(at, low, sum, number);
    sum = wave_sum64(sum);
    number = lane32(wave_scan32(number), 63);
    if (s.lane == 0) shared.part[s.wave] = sum, shared.ties[s.wave] = number;
    __syncthreads();
    // lane q of 16: wave q's weight, its tokens of the border taken in order
    const uint32_t most = (uint32_t)min(n, (uint64_t)0xffffffffu), q_ties = shared.ties[s.lane & 15];
    const uint32_t q_earlier = row_scan32(q_ties) - q_ties;
    const uint64_t q_mine = shared.part[s.lane & 15] + min(q_ties, most - min(most, q_earlier)) * one;
    const uint64_t q_upto = row_scan64(q_mine);
    const uint64_t total = lane64(q_upto, 15), mine = lane64(q_mine, s.wave);
    uint64_t before = lane64(q_upto, s.wave) - mine;
    uint32_t left_here = most - min(most, lane32(q_earlier, s.wave));
    const double f = u > 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
    const uint64_t aim = (uint64_t)(f * (double)total);
    if (before <= aim && aim < before + mine) {  // one wave, all of it
#pragma unroll 1
      for (int q = 0; q < s.chunks; ++q) {
        const uint32_t same = one ? shared.same[q][threadIdx.x] : 0, upto = wave_scan32(same);
        const uint32_t earlier = upto - same;  // the border's tokens before this lane's
        const uint32_t still = left_here - min(left_here, earlier);
        const uint64_t w = shared.own[q][threadIdx.x] + min(still, same) * one;
        const uint64_t to = before + wave_scan64(w);
        before = lane64(to, 63);
        left_here -= min(left_here, lane32(upto, 63));
        if (aim >= before) continue;
        const u32x4 raw = s.load(q);
        const bool by_table = tables && s.held(raw, at);
        // the lane that has it: its eight logits to eight lanes, lane e with the sum up to the e-th
        const int l = __builtin_ctzll(__ballot(aim < to));
        const u32x4 its = {lane32(raw[0], l), lane32(raw[1], l), lane32(raw[2], l), lane32(raw[3], l)};
        const int e = s.lane & 7;
        const uint32_t word = e < 4 ? (e < 2 ? its[0] : its[1]) : (e < 6 ? its[2] : its[3]);
        const uint32_t key = (e & 1 ? ordered2<T>(word) >> 16 : ordered2<T>(word)) & 0xffffu;
        const uint32_t tie = row_scan32(s.lane < 8 && key - low <= at - low && low <= at);
        uint64_t sum_e;
        if (by_table) {
          double part = 0x1p52;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            part = s.table_add(part, S::half(its[j >> 1], j), j <= e && S::half(ordered2<T>(its[j >> 1]), j) > at);
          sum_e = __builtin_bit_cast(uint64_t, part) & 0xfffffffffffffull;
        } else {
          sum_e = row_scan64(s.lane < 8 && key > at ? s.weight(key) : 0);
        }
        sum_e += lane64(to - w, l) + min(tie, lane32(still, l)) * one;
        const uint64_t past = __ballot(aim < sum_e) & 0xff;
        if (s.lane == 0) a.ids[r] = s.index(q) + 8 * l + __builtin_ctzll(past);
        break;
      }
    }
  }
}

}  // namespace atma

extern "C" int64_t atma_sample_tokens_workspace(int64_t rows, int64_t V, int dtype) {
  using namespace atma;
  if (rows < 1 || V < 1 || V > (1 << 20) || !dtype_size(dtype)) return 0;
  const int parts = wide_parts(rows, V, dtype);
  return parts ? rows * WideRow::bytes(parts, (int)((V + kSampleChunk - 1) / kSampleChunk)) : 0;
}

extern "C" int atma_sample_tokens_in(const void* logits, int64_t ld, const float* uniform, const float* temperature, float t0,
                                     const int32_t* top_k, int k0, const float* top_p, float p0, const float* min_p, float m0,
                                     int64_t* ids, int64_t rows, int64_t V, int dtype, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  using namespace atma;
  const char* what = "sample_tokens";
  if (!dtype_size(dtype)) return set_error(ATMA_ERR_UNSUPPORTED, "%s: fp32 or 16-bit logits (dtype %d)", what, dtype);
  if (rows < 0 || V < 1 || V > (1 << 20))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: 1 to 2^20 logits a row (rows=%lld V=%lld)", what, (long long)rows, (long long)V);
  if (rows == 0) return ATMA_OK;
  if (!logits || !uniform || !ids) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)logits % dtype_size(dtype)) return set_error(ATMA_ERR_INVALID, "%s: misaligned logits", what);
  if (rows > 1 && ld < V && ld != 0) return set_error(ATMA_ERR_INVALID, "%s: rows overlap", what);
  SampleArgs a{logits, ld, uniform, temperature, top_k, top_p, min_p, t0, p0, m0, k0, ids, (int)V, nullptr, 0};
  const int64_t need = atma_sample_tokens_workspace(rows, V, dtype);
  if (need && workspace) {
    if (workspace_bytes < need || (uintptr_t)workspace % 8)
      return set_error(ATMA_ERR_INVALID, "%s: a workspace of %lld bytes, 8-byte aligned", what, (long long)need);
    a.held = (uint8_t*)workspace;
    a.parts = wide_parts(rows, V, dtype);
    const dim3 grid((unsigned)a.parts, (unsigned)rows);
    hipStream_t st = (hipStream_t)stream;
    auto launch = [&](auto zero) {
      using T = decltype(zero);
      wide_top_kernel<T><<<grid, 512, 0, st>>>(a);
      const bool count = top_k || (k0 > 0 && k0 < V);
      if (count || top_p || p0 < 1.f) wide_bins_kernel<T><<<grid, 512, 0, st>>>(a);
      if (count) wide_list_kernel<T><<<grid, 512, 0, st>>>(a);
      wide_sums_kernel<T><<<grid, 512, 0, st>>>(a);
      wide_pick_kernel<T><<<dim3((unsigned)rows), 512, 0, st>>>(a);
    };
    if (dtype == ATMA_F32) launch(0.f);
    else if (dtype == ATMA_BF16) launch(bf16{});
    else launch(f16{});
    return check_launch(what);
  }
  // Short rows take workgroups of four waves, of which a CU holds five: us in bf16, four waves / values counted / sixteen waves, 32 rows of
  // 2,000 logits 12.9 / 14.7 / -, of 8,000 24.4 / 17.0 / 19.4 (eight), of 16,000 - / 19.2 / 25.0; 2,048 rows of 1,000 29 / 109 / -,
  // of 8,000 63 / 122 / 82 (eight), of 12,000 - / 131 / 155
  const bool small = V <= (rows > device_cu_count() ? 16384 : 4096);
  // a workgroup a row; a launch holds fewer than 2^32 threads, so what no one launch holds goes in several
  constexpr int64_t most = 1 << 20;
  for (int64_t r = 0; r < rows; r += most) {
    SampleArgs p = a;
    p.logits = (const char*)logits + r * ld * dtype_size(dtype);
    p.uniform += r;
    if (temperature) p.temperature += r;
    if (top_k) p.top_k += r;
    if (top_p) p.top_p += r;
    if (min_p) p.min_p += r;
    p.ids += r;
    const unsigned grid = (unsigned)std::min(rows - r, most);
    hipStream_t st = (hipStream_t)stream;
    auto launch = [&](auto zero) {
      using T = decltype(zero);
      if (small) {
        sample_tokens_kernel<T, 4><<<grid, 256, 0, st>>>(p);
        return;
      }
      if constexpr (sizeof(T) == 2) {
        if (V < 65536) {
          sample_counted_kernel<T><<<grid, kCountedThreads, 0, st>>>(p);
          return;
        }
      }
      sample_tokens_kernel<T, 16><<<grid, 1024, 0, st>>>(p);
    };
    if (dtype == ATMA_BF16) launch(bf16{});
    else if (dtype == ATMA_F16) launch(f16{});
    else launch(float{});
  }
  return check_launch(what);
}

extern "C" int atma_sample_tokens(const void* logits, int64_t ld, const float* uniform, const float* temperature, float t0,
                                  const int32_t* top_k, int k0, const float* top_p, float p0, const float* min_p, float m0,
                                  int64_t* ids, int64_t rows, int64_t V, int dtype, void* stream) {
  return atma_sample_tokens_in(logits, ld, uniform, temperature, t0, top_k, k0, top_p, p0, min_p, m0, ids, rows, V, dtype, nullptr,
                               0, stream);
}
