// What the tiled products with 8-bit and 4-bit weights (fp8_gemm.hip, fp4_gemm.hip) share: the order of the tiles, copies of
// single words and bytes into LDS, biases, stores and the choice of a tile.
#pragma once

#include <math.h>

#include <algorithm>

#include "common.h"

namespace atma {

__device__ __forceinline__ float bias_f32(int dtype, uint32_t bits) {
  if (dtype == ATMA_F32) return __builtin_bit_cast(float, bits);
  const uint16_t v = (uint16_t)bits;
  return dtype == ATMA_BF16 ? to_f32(__builtin_bit_cast(bf16, v)) : to_f32(__builtin_bit_cast(f16, v));
}

// Outputs n0 .. n0 + 7 of a row that ends at N.  Rows of odd widths start at any element: the vector stores take any address
// (elements one by one cost 184 us instead of 109 at 28,106 x 1,712 -> 1,557); whole: the
// tile has every feature
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
__device__ __forceinline__ void store_out8(uint16_t* y, const u32x4& o, bool whole, int64_t n0, int64_t N) {
  if (whole || n0 + 8 <= N) {
    *(u32x4_any*)y = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n0 + e < N) y[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
  }
}

// relu(a)^2 * gate in fp32 (v_maximum3_f32: NaN passes through, as torch's relu)
__device__ __forceinline__ float gate_act(float av, float gv) {
  const float pos = __builtin_elementwise_maximum(av, 0.f);
  return gv * (pos * pos);
}

// Rows of 128 bytes in LDS, eight chunks of 16, chunk c of row r at position c ^ x_swizzle(r): the 16 lanes that read one chunk
// of 16 rows cover all banks when it takes eight values over the rows of each parity
__device__ __forceinline__ int x_swizzle(int r) { return (r >> 1) & 7; }

// The 4-byte copy where a descriptor may just have been read back from a vector register: five wait states before it
__device__ __forceinline__ void dma_buf4_rare(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds_byte_offset) {
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(r),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds_byte_offset))
               : "memory");
}
// A byte a lane, from an address a lane, to the word at lds_byte_offset + 4 lane
__device__ __forceinline__ void dma_load1_at(const void* p, uint32_t lds_byte_offset) {
  asm volatile("s_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(p),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds_byte_offset))
               : "memory");
}

// Two bytes, or a word, a lane, likewise
__device__ __forceinline__ void dma_load2_at(const void* p, uint32_t lds_byte_offset) {
  asm volatile("s_nop 0\n\tglobal_load_lds_ushort %0, off" ::"v"(p),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds_byte_offset))
               : "memory");
}
__device__ __forceinline__ void dma_load4_at(const void* p, uint32_t lds_byte_offset) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds_byte_offset))
               : "memory");
}

// Tile u of an XCD: each owns a contiguous range, walked as groups of four token tiles x all feature tiles
template <typename C, typename A>
__device__ __forceinline__ bool gemm_tile_at(const A& a, int xcd, int u, int64_t& m0, int64_t& f0) {
  const int t = xcd * a.per_xcd + u;
  if (u >= a.per_xcd || t >= a.m_tiles * a.f_tiles) return false;
  const int grp = t / (4 * a.f_tiles), r = t - grp * 4 * a.f_tiles;
  const int gm = min(4, a.m_tiles - 4 * grp);
  m0 = (int64_t)(4 * grp + r % gm) * C::BM;
  f0 = (int64_t)(r / gm) * C::OF;
  return true;
}

// What a tile shape costs: us a tile to begin and end it, and us a block of K, where few CUs work (latency) and where all do
struct TileCost {
  int features, tokens;
  float tile, few, all;
};

inline float tile_time(int64_t M, int64_t N, int nk, const TileCost& c) {
  const int64_t tiles = ((M + c.tokens - 1) / c.tokens) * ((N + c.features - 1) / c.features);
  const float fill = (float)tiles / (float)device_cu_count();
  if (fill <= 1.f) return c.tile + (float)nk * (c.few + (c.all - c.few) * fill);
  return ceilf(fill) * (c.tile + (float)nk * c.all);
}

inline int cheapest_tile(int64_t M, int64_t N, int nk, const TileCost* c, int n) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < n; ++i) {
    const float t = tile_time(M, N, nk, c[i]);
    if (i == 0 || t < least) best = i, least = t;
  }
  return best;
}

}  // namespace atma
