// Block-scaled 8-bit products: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]) for x (M, K) with a scale for each 128 values of
// a row and w (N, K) with a scale for each 128 x 128 block (fp8.h), and the MLP's first projection with its activation
// formed from the fp32 sums, h = gate * relu(a)^2, and quantized in the epilogue.  No reference counterpart.
//
// Products: v_mfma_scale_f32_32x32x64_f8f6f4, two for each block of 128 along K (few rows: 16x16x128, one).  Its scale
// operands carry the blocks' power-of-two scales, a lane its row's, so the accumulator holds scaled sums from the first product
// on and no partial sum is ever rescaled.  Accumulators are fp32; inside the instruction the products of eight neighbouring k
// are aligned to the largest of them and keep about 14 bits below it (measured: 2^2 beside 2^16 is lost), which is 1.4e-5
// of the result for normally distributed values: far below the rounding to a 16-bit output, and the reason why there is
// no fp32 output.  The order of k inside a block is free (one scale covers it), so a lane takes whichever 16-byte pieces
// load best, the same ones of x and w.
#include <math.h>

#include <algorithm>

#include "fp8.h"

namespace atma {

typedef int i32x8 __attribute__((ext_vector_type(8)));

union Frag8 {  // one operand: 32 values of a row
  i32x8 v;
  u32x4 q[2];
};

struct Fp8Args {
  const uint8_t* x;  // (M, K), row stride ldx
  int64_t ldx;
  const uint8_t* xs;  // (M, nk), row stride ldxs
  int64_t ldxs;
  const uint8_t* w;  // (N, K) or, gated, (2 N, K): the a rows, then the gate rows
  int64_t ldw;
  const uint8_t* ws;  // (ceil(rows / 128), nk), row stride ldws
  int64_t ldws;
  int64_t w_blocks;  // rows of ws
  const void* bias;  // (N,) or (2 N,), or null
  int bias_dtype;
  void* y;  // (M, N): T, or gated: e4m3fn
  int64_t ldy;
  uint8_t* ys;  // gated: the output's scales (M, N / 128), row stride ldys
  int64_t ldys;
  int64_t M, N;
  int K, nk;
  int m_tiles, f_tiles, per_xcd;
};

// The biases of features n .. n + 3 as their bits, in loads of their own size (nothing behind the last of `rows` is read;
// features past it read as the last), converted where they are added: nothing waits for them here
struct BiasBits {
  uint32_t w[4];
  uint16_t v[4];
};
__device__ __forceinline__ BiasBits bias_load(const Fp8Args& a, int64_t n, int64_t rows) {
  const void* p = a.bias ? a.bias : a.w;
  BiasBits b;
  if (a.bias_dtype == ATMA_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) b.w[e] = ((const uint32_t*)p)[min(n + e, rows - 1)];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) b.v[e] = ((const uint16_t*)p)[min(n + e, rows - 1)];
  }
  return b;
}
__device__ __forceinline__ float bias_f32(int dtype, uint32_t bits) {
  if (dtype == ATMA_F32) return __builtin_bit_cast(float, bits);
  const uint16_t v = (uint16_t)bits;
  return dtype == ATMA_BF16 ? to_f32(__builtin_bit_cast(bf16, v)) : to_f32(__builtin_bit_cast(f16, v));
}
__device__ __forceinline__ float bias_value(const Fp8Args& a, const BiasBits& b, int e) {
  return a.bias ? bias_f32(a.bias_dtype, a.bias_dtype == ATMA_F32 ? b.w[e] : b.v[e]) : 0.f;
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

// Rows of 128 bytes in LDS, eight chunks of 16, chunk c of row r at position c ^ f(r): the 16 lanes that read one chunk of
// 16 rows cover all banks when f takes eight values over the rows of each parity (65,536 x 1,024 -> 4,096 gated: 0 of 6.0e7 LDS
// cycles are conflicts; tiles of 16 tokens a wave lose 5% to their scales, which lie 256 bytes apart).  The weights are
// the MFMA's rows, in an order such that a lane's accumulators are 16 consecutive features of one token (row 8 q + 4 h + e
// is feature 16 h + 4 q + e; lane half h holds the rows 4 h + e of each 8): outputs are stored straight from registers.
__device__ __forceinline__ int x_swizzle(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int w_swizzle(int r) { return ((r >> 1) & 3) | (((r >> 4) & 1) << 2); }

// The kernel's arguments read again where they are needed: kept in scalar registers through the loop they would be spilled
typedef const __attribute__((address_space(4))) Fp8Args* LateArgs;
__device__ __forceinline__ LateArgs late_args() {
  LateArgs p = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

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

// Tile u of an XCD: each owns a contiguous range, walked as groups of four token tiles x all feature tiles
template <typename C, typename A>
__device__ __forceinline__ bool fp8_tile_at(const A& a, int xcd, int u, int64_t& m0, int64_t& f0) {
  const int t = xcd * a.per_xcd + u;
  if (u >= a.per_xcd || t >= a.m_tiles * a.f_tiles) return false;
  const int grp = t / (4 * a.f_tiles), r = t - grp * 4 * a.f_tiles;
  const int gm = min(4, a.m_tiles - 4 * grp);
  m0 = (int64_t)(4 * grp + r % gm) * C::BM;
  f0 = (int64_t)(r / gm) * C::OF;
  return true;
}

__device__ __forceinline__ f32x4 mfma_fp8(const Frag8& w, const Frag8& x, const f32x4& c, int ws, int xs) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, c, 0, 0, 0, ws, 0, xs);
}

// ------------------------------------------------------------------------------------------------ tiles
// A workgroup of WF x WM waves owns BF weight rows x BM tokens, a wave TF x TM tiles of 32 x 32
// (v_mfma_scale_f32_32x32x64_f8f6f4: two instructions for a block of 128 along K).  K runs in blocks through a ring of NS
// stages in LDS, filled by direct copies of whole 128-byte lines (a CU takes in 58 to 94 bytes a cycle that way, 29 to 54
// in rows of 64 bytes: measured from L2 with four and eight waves).  While the products of one half of a block run from
// registers, the operands of the next half are read from LDS, a token operand into the registers of the one just used,
// the weights into a second set; in the second half the copies of block k + NS go into the stage just read.  The
// workgroup is persistent and all of this runs on across its tiles: a tile's first copies fly and its first operands are
// read during the last blocks of the one before.
//
// A block is straight code (the compiler gathers products behind any branch): copies behind the last tile go on, out of
// range, and the scales of a block come with its copies.
template <int TF, int TM, int WF, int WM, int NS_, bool GATED>
struct Fp8Tile {
  static constexpr int NW = WF * WM, NS = NS_;
  static constexpr int BF = 32 * TF * WF, BM = 32 * TM * WM;
  static constexpr int OF = GATED ? BF / 2 : BF;  // output features
  static constexpr int TO = GATED ? TF / 2 : TF;  // tiles of output features a wave
  static constexpr int STAGE = (BF + BM) * kFp8Block;
  static constexpr int WCOPY = BF / 8 / NW, XCOPY = BM / 8 / NW, COPIES = WCOPY + XCOPY;  // a wave and block, 8 rows each
  static constexpr int XW = BM / NW;     // token scales a wave copies
  static constexpr int RING = NS + 2;    // blocks and tiles under way: copies run NS blocks ahead
  static constexpr int SLOT = NW * 256;  // a block's scales
  static constexpr int AUX = NS * STAGE, BIAS = AUX + RING * SLOT, TOP = BIAS + RING * 1024;
  static constexpr bool TURNED = !GATED && NW == 8;  // outputs leave through LDS, where there is room
  static constexpr int TURN = TOP, LDS = TOP + (GATED ? WF * BM * 4 : TURNED ? 2048 * NW : 0);
  static_assert((NW == 4 || NW == 8) && BF % (8 * NW) == 0 && BM % (8 * NW) == 0 && BF <= 256 && XW <= 32,
                "whole copies, a bias of 1 KiB");
  static_assert(!GATED || (OF == kFp8Block && TF == 2), "a gated tile is one block of output features");
  static_assert((NS - 2) * (COPIES + 1) < 63, "vmcnt counts to 63");
};

template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED>
__global__ void __launch_bounds__(64 * WF * WM, 2) fp8_tile_kernel(Fp8Args a) {
  using C = Fp8Tile<TF, TM, WF, WM, NS, GATED>;
  constexpr int TO = C::TO;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wm = wave / WF;
  const int r = lane & 31, h = lane >> 5;
  const int nk = a.nk;
  int64_t m0, f0;
  int u = blockIdx.x >> 3;
  if (!fp8_tile_at<C>(a, blockIdx.x & 7, u, m0, f0)) return;

  // ---- the copies, NS blocks ahead.  Copy i of a wave moves rows 8 (i NW + wave) .. + 7: lane l writes row l / 8,
  // position l % 8, and reads the chunk that belongs there; out of range (chunks past K, rows past the end, everything
  // behind the last tile) zeros are written
  const uint32_t lds0 = lds_offset(lds);
  const int crow = 8 * wave + (lane >> 3);
  const int wk = 16 * ((lane & 7) ^ w_swizzle(crow)), xk = 16 * ((lane & 7) ^ x_swizzle(crow));
  const uint32_t wv0 = (uint32_t)crow * (uint32_t)a.ldw + (uint32_t)wk, xv0 = (uint32_t)crow * (uint32_t)a.ldx + (uint32_t)xk;
  const uint32_t wstep = 8u * C::NW * (uint32_t)a.ldw, xstep = 8u * C::NW * (uint32_t)a.ldx;
  __amdgpu_buffer_rsrc_t xr, wr, gr;
  const uint8_t* scales;  // a lane's row: lanes 0 .. XW - 1 token rows, 32 and 33 weight blocks, the others as lane 0
  int pu = u, pk = 0, plimit = 0, ptile = 0, pslot = 0, pstage = 0;
  auto aim = [&](int64_t tm0, int64_t tf0) {
    LateArgs p = late_args();
    const int64_t rows = min((int64_t)C::BM, p->M - tm0);
    xr = buffer_rsrc(p->x + tm0 * p->ldx, (uint32_t)(rows * p->ldx));
    const uint32_t wb = (uint32_t)(min((int64_t)C::OF, p->N - tf0) * p->ldw);
    wr = buffer_rsrc(p->w + tf0 * p->ldw, wb);
    if constexpr (GATED) gr = buffer_rsrc(p->w + (p->N + tf0) * p->ldw, wb);
    const int64_t m = min(tm0 + C::XW * wave + (lane < C::XW ? lane : 0), p->M - 1);
    const int64_t b0 = tf0 / kFp8Block;
    const int64_t b = lane == 33 ? (GATED ? b0 + p->N / kFp8Block : min(b0 + 1, p->w_blocks - 1)) : b0;
    scales = lane == 32 || lane == 33 ? p->ws + b * p->ldws : p->xs + m * p->ldxs;
    plimit = p->K;
    if (p->bias && wave == 2) {
      // the tile's biases (gated: 128 of a, 128 of gate), in whole words, to its slot
      const int size = p->bias_dtype == ATMA_F32 ? 4 : 2;
      const int64_t total = (GATED ? 2 : 1) * p->N * size;
      const __amdgpu_buffer_rsrc_t br = buffer_rsrc(p->bias, (uint32_t)total);
      for (int i = 0; i < size; ++i) {
        const int f = (64 * i + lane) * 4 / size;  // the word's first feature in the tile
        const int64_t n = tf0 + (GATED && f >= C::OF ? p->N + f - C::OF : f);
        dma_buf4_rare(br, n * size + 4 <= total ? (uint32_t)(n * size) : 0xfffffffcu,
                      lds0 + C::BIAS + 1024 * ptile + 256 * i);
      }
    }
    ptile = ptile + 1 == C::RING ? 0 : ptile + 1;
  };
  auto next_tile = [&]() {
    int64_t nm0, nf0;
    pk = 0;
    pu += gridDim.x >> 3;
    if (fp8_tile_at<C>(*late_args(), blockIdx.x & 7, pu, nm0, nf0)) aim(nm0, nf0);
    else plimit = 0;
  };
  uint32_t pd, pwv, pxv;
  auto copies_begin = [&]() {
    dma_load1_at(scales + (plimit ? pk : 0), lds0 + C::AUX + C::SLOT * pslot + 256 * wave);
    pslot = pslot + 1 == C::RING ? 0 : pslot + 1;
    pd = lds0 + pstage * C::STAGE + 1024 * wave;
    pstage = pstage + 1 == NS ? 0 : pstage + 1;
    const int k = kFp8Block * pk++;
    pwv = k + wk < plimit ? wv0 + (uint32_t)k : 0x80000000u;
    pxv = k + xk < plimit ? xv0 + (uint32_t)k : 0x80000000u;
  };
  auto copy = [&](int i) {
    constexpr int half = C::WCOPY / 2;  // gated: the first half of a wave's copies are a rows, the others gate rows
    if (i >= C::WCOPY) dma_buf16_at(xr, pxv + (i - C::WCOPY) * xstep, 0u, pd + C::BF * kFp8Block + 1024 * C::NW * (i - C::WCOPY));
    else if (GATED && i >= half) dma_buf16_at(gr, pwv + (i - half) * wstep, 0u, pd + 1024 * C::NW * i);
    else dma_buf16_at(wr, pwv + i * wstep, 0u, pd + 1024 * C::NW * i);
  };

  // ---- operand reads: half s of a block is the chunks 4 s .. 4 s + 3, lane half h takes two of them
  const int wrow0 = 32 * TO * wf;  // the wave's first output feature in the tile
  const int wrow = 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
  uint32_t wofs[2][2], xofs[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      wofs[s][q] = (uint32_t)((wrow0 + wrow) * kFp8Block + 16 * ((4 * s + 2 * h + q) ^ w_swizzle(wrow)));
      xofs[s][q] = (uint32_t)((C::BF + 32 * TM * wm + r) * kFp8Block + 16 * ((4 * s + 2 * h + q) ^ x_swizzle(r)));
    }
  auto wtile = [](int t) { return GATED ? t / TO * (C::BF / 2) + 32 * (t % TO) : 32 * t; };
  f32x16 acc[TF][TM];
  Frag8 wv[2][TF], xv[TM];
  int xs[TM], ws[2];
  int stage = 0, slot = 0, tile = 0;  // what is read next
  auto read_w = [&](const uint8_t* base, int s, int t) {
#pragma unroll
    for (int q = 0; q < 2; ++q) wv[s][t].q[q] = *(const u32x4*)(base + wofs[s][q] + kFp8Block * wtile(t));
  };
  auto read_x = [&](const uint8_t* base, int s, int j) {
#pragma unroll
    for (int q = 0; q < 2; ++q) xv[j].q[q] = *(const u32x4*)(base + xofs[s][q] + kFp8Block * 32 * j);
  };
  auto read_scales = [&]() {
    const uint8_t* p = lds + C::AUX + C::SLOT * slot;
    slot = slot + 1 == C::RING ? 0 : slot + 1;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int row = 32 * (TM * wm + j) + r;
      xs[j] = *(const int*)(p + 256 * (row / C::XW) + 4 * (row % C::XW));
    }
    const int* q = (const int*)(p + 256 * wave + 128);
    ws[0] = q[GATED ? 0 : wrow0 / kFp8Block];
    ws[1] = GATED ? q[1] : 0;
  };

  aim(m0, f0);
#pragma unroll 1
  for (int i = 0; i < NS; ++i) {
    if (pk == nk) next_tile();
    copies_begin();
#pragma unroll
    for (int c = 0; c < C::COPIES; ++c) copy(c);
  }
  wait_vmcnt<(NS - 1) * (C::COPIES + 1)>();
  lds_barrier();
#pragma unroll
  for (int t = 0; t < TF; ++t) read_w(lds, 0, t);
#pragma unroll
  for (int j = 0; j < TM; ++j) read_x(lds, 0, j);
  read_scales();
  while (true) {
    // ---- the sums start from the bias
#pragma unroll
    for (int t = 0; t < TF; ++t) {
      float b[16] = {};
      const int f = wrow0 + 16 * h + (GATED ? t / TO * C::OF + 32 * (t % TO) : 32 * t);
      LateArgs p = late_args();
      if (p->bias) {
        const uint8_t* at = lds + C::BIAS + 1024 * tile;
        if (p->bias_dtype == ATMA_F32) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const f32x4 v = *(const f32x4*)(at + 4 * (f + e));
            b[e] = v[0], b[e + 1] = v[1], b[e + 2] = v[2], b[e + 3] = v[3];
          }
        } else {
          if (!GATED && t == 0 && p->N % 2 && f0 + C::OF >= p->N) {
            // the last of an odd number is half a word, which no copy brings: every wave puts it beside the others
            *(uint16_t*)(lds + C::BIAS + 1024 * tile + 2 * (int)(p->N - 1 - f0)) = ((const uint16_t*)p->bias)[p->N - 1];
            wave_sync();
          }
          const bool bf = p->bias_dtype == ATMA_BF16;
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            const u32x4 v = *(const u32x4*)(at + 2 * (f + e));
#pragma unroll
            for (int i = 0; i < 8; ++i) b[e + i] = bf ? elem16<bf16>(v, i) : elem16<f16>(v, i);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][j][e] = b[e];
    }
    tile = tile + 1 == C::RING ? 0 : tile + 1;

    for (int kb = 0; kb < nk; ++kb) {
      if (pk == nk) next_tile();
      const uint8_t* base = lds + stage * C::STAGE;
      stage = stage + 1 == NS ? 0 : stage + 1;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s == 1) {
          // the next block's copies have landed in every wave, and every wave has read this block
          wait_vmcnt<(NS - 2) * (C::COPIES + 1)>();
          lds_barrier();
          base = lds + stage * C::STAGE;
          copies_begin();
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = 0; t < TF; ++t)
            acc[t][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                wv[s][t].v, xv[j].v, acc[t][j], 0, 0, 0, ws[GATED ? t / TO : 0], 0, xs[j]);
          // behind the products of token tile j: its operand of the next half, a share of the weights and copies
          read_x(base, s ^ 1, j);
#pragma unroll
          for (int t = j * TF / TM; t < (j + 1) * TF / TM; ++t) read_w(base, s ^ 1, t);
          if (s == 1) {
#pragma unroll
            for (int c = j * C::COPIES / TM; c < (j + 1) * C::COPIES / TM; ++c) copy(c);
            if (j == TM - 1) read_scales();
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- epilogue of tile (m0, f0): token 32 (TM wm + j) + r, 16 consecutive features a tile
    LateArgs p = late_args();
    if constexpr (!GATED) {
      const bool whole = f0 + C::OF <= p->N;  // every feature of the tile
      if constexpr (C::TURNED) {
        // through LDS, a wave its own 2 KiB: 32 tokens x 32 features at a time turn from a token a lane to 64-byte pieces, four
        // lanes each (chunk c of row r at position c ^ (r / 4) % 4): a CU alone stores 80 bytes a cycle so, 28 as they lie
        // (65,536 x 1,024 -> 8,192 630 to 605 us, 4,096 x 1,024 -> 4,096 23.4 to 21.8)
        uint8_t* turn = lds + C::TURN + 2048 * wave;
        const int64_t ldy = p->ldy, N = p->N, M = p->M;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
          for (int t = 0; t < TF; ++t) {
            const f32x16& v = acc[t][j];
            wave_sync();
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              *(u32x4*)(turn + 64 * r + 16 * ((2 * h + e / 8) ^ ((r >> 2) & 3))) =
                  u32x4{pack2<T>(v[e], v[e + 1]), pack2<T>(v[e + 2], v[e + 3]), pack2<T>(v[e + 4], v[e + 5]),
                        pack2<T>(v[e + 6], v[e + 7])};
            wave_sync();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int row = 16 * i + (lane >> 2);
              const u32x4 o = *(const u32x4*)(turn + 64 * row + 16 * ((lane & 3) ^ ((row >> 2) & 3)));
              const int64_t m = m0 + 32 * (TM * wm + j) + row, n0 = f0 + wrow0 + 32 * t + 8 * (lane & 3);
              if (m < M) store_out8((uint16_t*)p->y + m * ldy + n0, o, whole, n0, N);
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int64_t m = m0 + 32 * (TM * wm + j) + r;
          if (m < p->M) {
#pragma unroll
            for (int t = 0; t < TF; ++t) {
              const int64_t n0 = f0 + wrow0 + 32 * t + 16 * h;
              const f32x16& v = acc[t][j];
#pragma unroll
              for (int e = 0; e < 16; e += 8)
                store_out8((uint16_t*)p->y + m * p->ldy + n0 + e,
                           u32x4{pack2<T>(v[e], v[e + 1]), pack2<T>(v[e + 2], v[e + 3]), pack2<T>(v[e + 4], v[e + 5]),
                                 pack2<T>(v[e + 6], v[e + 7])},
                           whole, n0 + e, p->N);
            }
          }
        }
      }
    } else {
      // the activations in place of a's sums, their largest magnitude over the wave's features, then over the tile's
      float* part = (float*)(lds + C::TOP);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = gate_act(acc[0][j][e], acc[1][j][e]);
          acc[0][j][e] = v;
          top = fmaxf(top, fabsf(v));
        }
        if (top == __builtin_inff()) {  // (NaN does not enter the maximum; infinities must not)
          top = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, finite_abs(acc[0][j][e]));
        }
        top = fmaxf(top, wave_xor(top, 32));
        if (h == 0) part[wf * C::BM + 32 * (TM * wm + j) + r] = top;
      }
      lds_barrier();
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int row = 32 * (TM * wm + j) + r;
        float top = part[row];
#pragma unroll
        for (int q = 1; q < WF; ++q) top = fmaxf(top, part[q * C::BM + row]);
        const int code = fp8_scale_code(top);
        const float scale = fp8_scale(code);
        const int64_t m = m0 + row;
        if (m < p->M) {
          if (wf == 0 && h == 0) p->ys[m * p->ldys + f0 / kFp8Block] = (uint8_t)code;
          const f32x16& v = acc[0][j];
          u32x4 o;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            o[q] = fp8_scaled4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3], scale);
          *(u32x4*)((uint8_t*)p->y + m * p->ldy + f0 + wrow0 + 16 * h) = o;
        }
      }
    }
    u += gridDim.x >> 3;
    if (!fp8_tile_at<C>(*late_args(), blockIdx.x & 7, u, m0, f0)) break;
  }
  wait_vmcnt<0>();  // no copy outlives its workgroup's LDS
}

// ------------------------------------------------------------------------------------------------ few rows
// Few rows: latency, not bandwidth.  A workgroup owns FT tiles of 16 features x MT tiles of 16 tokens and its NW waves take the
// blocks of K in turn, so a chain of K is NW times shorter; their sums are joined through LDS in a fixed order.  Each wave
// has a ring of its own of NS blocks, filled by direct copies of whole 128-byte lines, and waits for nothing but its own
// copies.  Operands read from memory in the MFMA's layout, 16 rows to an instruction, come in at 28 GB/s a CU, at 46 with
// the halves of odd rows swapped, copied this way at 104 (64 x 16,384 -> 1,024 30.7, 20.6 and 10.5 us).  The bias is read
// ahead of the sums (0.25 to 0.3 us).  Four waves of two blocks measured best: more waves or more copies in flight leave fewer
// workgroups a CU (32 x 1,024 -> 1,024, 8 waves 3.7 us, 4 waves of four blocks 3.6, of two 3.2).
template <typename T, int MT, int FT, int NW, int NS>
__global__ void __launch_bounds__(64 * NW) fp8_few_kernel(Fp8Args a) {
  constexpr int ROWS = 16 * (FT + MT), STAGE = ROWS * kFp8Block + 256, COPIES = ROWS / 8;
  static_assert(FT * MT <= NW && FT * MT * 1024 <= NS * STAGE && 16 * MT < 64 && kFp8Block % (16 * FT) == 0,
                "the sums fit the ring, a lane is left for the weights' scale, one block of weight rows");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NW * NS * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 16 * FT, m0 = (int64_t)blockIdx.y * 16 * MT;
  const __amdgpu_buffer_rsrc_t wr = buffer_rsrc(a.w + f0 * a.ldw, (uint32_t)(min((int64_t)16 * FT, a.N - f0) * a.ldw));
  const __amdgpu_buffer_rsrc_t xr = buffer_rsrc(a.x + m0 * a.ldx, (uint32_t)(min((int64_t)16 * MT, a.M - m0) * a.ldx));
  // copy i of a block moves rows 8 i .. 8 i + 7, lane l the chunk that belongs at position l % 8 of row 8 i + l / 8
  const int crow = lane >> 3, chunk = 16 * ((lane & 7) ^ (crow >> 1));
  const uint32_t wv0 = (uint32_t)crow * (uint32_t)a.ldw, xv0 = (uint32_t)crow * (uint32_t)a.ldx;
  const uint8_t* scales = lane < 16 * MT ? a.xs + min(m0 + lane, a.M - 1) * a.ldxs : a.ws + f0 / kFp8Block * a.ldws;
  uint8_t* ring = lds + wave * NS * STAGE;
  const uint32_t ring0 = lds_offset(ring);
  auto copies = [&](int kk, int slot) {
    const uint32_t d = ring0 + slot * STAGE;
    dma_load1_at(scales + min(kk, a.nk - 1), d + ROWS * kFp8Block);
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int k = kk * kFp8Block + (chunk ^ (i % 2 * 64));  // (K <= 2^22: no overflow in the blocks behind the last)
      const bool w = i < 2 * FT;
      const uint32_t at = w ? wv0 + 8u * i * (uint32_t)a.ldw : xv0 + 8u * (i - 2 * FT) * (uint32_t)a.ldx;
      dma_buf16_at(w ? wr : xr, k < a.K ? at + (uint32_t)k : 0x80000000u, 0u, d + 1024 * i);
    }
  };
#pragma unroll
  for (int i = 0; i < NS; ++i) copies(wave + i * NW, i);
  // the output tile that the wave joins
  const int ot = wave / MT, oj = wave % MT;
  const int64_t n0 = f0 + 16 * ot + 4 * g, m = m0 + 16 * oj + r;
  const BiasBits bias = bias_load(a, n0, a.N);
  f32x4 acc[FT][MT] = {};
  int slot = 0;
  for (int kk = wave; kk < a.nk; kk += NW) {
    wait_vmcnt<(NS - 1) * (COPIES + 1)>();
    const uint8_t* base = ring + slot * STAGE;
    Frag8 wv[FT], xv[MT];
    int xsc[MT];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = r * kFp8Block + 16 * ((4 * q + g) ^ x_swizzle(r));
#pragma unroll
      for (int t = 0; t < FT; ++t) wv[t].q[q] = *(const u32x4*)(base + 2048 * t + at);
#pragma unroll
      for (int j = 0; j < MT; ++j) xv[j].q[q] = *(const u32x4*)(base + 2048 * (FT + j) + at);
    }
    const int* sc = (const int*)(base + ROWS * kFp8Block);
#pragma unroll
    for (int j = 0; j < MT; ++j) xsc[j] = sc[16 * j + r];
    const int wsc = sc[16 * MT];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the copies that overwrite them start
    copies(kk + NS * NW, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[t][j] = mfma_fp8(wv[t], xv[j], acc[t][j], wsc, xsc[j]);
  }
  wait_vmcnt<0>();
  __syncthreads();  // every wave's copies, those behind the last block too, are done: the ring is free
  auto red = (f32x4(*)[FT][MT][64])lds;
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[wave][t][j][lane] = acc[t][j];
  __syncthreads();
  if (wave >= FT * MT || m >= a.M) return;
  f32x4 s = red[0][ot][oj][lane];
#pragma unroll
  for (int q = 1; q < NW; ++q) s += red[q][ot][oj][lane];
  T* y = (T*)a.y + m * a.ldy + n0;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = s[e] + bias_value(a, bias, e);
  if (n0 + 4 <= a.N) {
    *(u32x2_any*)y = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n0 + e < a.N) y[e] = from_f32<T>(v[e]);
  }
}

// Few rows of the gated form: a workgroup owns one block of 128 output features, whose scale stays inside, x 16 tokens.  Each of
// its eight waves has 16 features, the a rows and the gate rows, all of K through a ring of the wave's own; the tokens come in
// once, all of K, before the first block.  Bound by the 32 KiB of weights a block that one CU takes in (0.25 us: 62 bytes a
// cycle) behind 3.2 us of launch, first copies and epilogue: us for 16 x 1,024 -> 4,096 and 16 x 4,096 -> 1,024, the 64-token
// tile 7.8 and 18.3, tokens in each wave's ring 6.9 and 17.0, this 5.4 and 11.2 (5.8 and 11.6 with the bias read at the end).
constexpr int kGatedFewBlocks = 36;  // of K, that LDS holds
__global__ void __launch_bounds__(512) fp8_gated_few_kernel(Fp8Args a) {
  constexpr int NS = 2, STAGE = 32 * kFp8Block, XB = 16 * kFp8Block + 256;  // a block of tokens, then its scales in words
  __shared__ __attribute__((aligned(1024))) uint8_t lds[8 * NS * STAGE + kGatedFewBlocks * XB];
  __shared__ float part[8][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * kFp8Block, m0 = (int64_t)blockIdx.y * 16, fb = blockIdx.x;
  const uint32_t wb = (uint32_t)(kFp8Block * a.ldw);
  const __amdgpu_buffer_rsrc_t ar = buffer_rsrc(a.w + f0 * a.ldw, wb), gr = buffer_rsrc(a.w + (a.N + f0) * a.ldw, wb);
  const __amdgpu_buffer_rsrc_t xr = buffer_rsrc(a.x + m0 * a.ldx, (uint32_t)(min((int64_t)16, a.M - m0) * a.ldx));
  // copies move 8 rows of 128 bytes as in fp8_few_kernel
  const int crow = lane >> 3, chunk = 16 * ((lane & 7) ^ (crow >> 1));
  const uint32_t wv0 = (uint32_t)(16 * wave + crow) * (uint32_t)a.ldw, xv0 = (uint32_t)crow * (uint32_t)a.ldx;
  const uint8_t* xs = lds + 8 * NS * STAGE;
  const uint32_t xs0 = lds_offset(xs);
  const uint8_t* scales = lane < 32 ? a.xs + min(m0 + r, a.M - 1) * a.ldxs
                                    : a.ws + (lane == 33 ? fb + a.N / kFp8Block : fb) * a.ldws;
  for (int kk = wave; kk < a.nk; kk += 8) {
    const uint32_t d = xs0 + kk * XB;
    dma_load1_at(scales + kk, d + 16 * kFp8Block);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = kk * kFp8Block + (chunk ^ (64 * i));
      dma_buf16_at(xr, k < a.K ? xv0 + 8u * i * (uint32_t)a.ldx + (uint32_t)k : 0x80000000u, 0u, d + 1024 * i);
    }
  }
  const uint8_t* ring = lds + wave * NS * STAGE;
  const uint32_t ring0 = lds_offset(ring);
  auto copies = [&](int kk, int slot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = kk * kFp8Block + (chunk ^ (i % 2 * 64));
      dma_buf16_at(i < 2 ? ar : gr, k < a.K ? wv0 + 8u * (i % 2) * (uint32_t)a.ldw + (uint32_t)k : 0x80000000u, 0u,
                   ring0 + slot * STAGE + 1024 * i);
    }
  };
#pragma unroll
  for (int i = 0; i < NS; ++i) copies(i, i);
  wait_vmcnt<4 * NS>();
  lds_barrier();  // the tokens are there, from every wave
  const int64_t n0 = f0 + 16 * wave + 4 * g, m = m0 + r;
  const BiasBits ba = bias_load(a, n0, 2 * a.N), bg = bias_load(a, a.N + n0, 2 * a.N);
  f32x4 acc[2] = {};
  int slot = 0;
  for (int kk = 0; kk < a.nk; ++kk) {
    wait_vmcnt<4 * (NS - 1)>();
    const uint8_t *wp = ring + slot * STAGE, *xp = xs + kk * XB;
    Frag8 wv[2], xv;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = r * kFp8Block + 16 * ((4 * q + g) ^ x_swizzle(r));
#pragma unroll
      for (int t = 0; t < 2; ++t) wv[t].q[q] = *(const u32x4*)(wp + 2048 * t + at);
      xv.q[q] = *(const u32x4*)(xp + at);
    }
    const int* sc = (const int*)(xp + 16 * kFp8Block);
    const int xsc = sc[r], wsc[2] = {sc[32], sc[33]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the copies that overwrite them start
    copies(kk + NS, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[t] = mfma_fp8(wv[t], xv, acc[t], wsc[t], xsc);
  }
  wait_vmcnt<0>();  // no copy outlives its workgroup's LDS
  f32x4 h;
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = gate_act(acc[0][e] + bias_value(a, ba, e), acc[1][e] + bias_value(a, bg, e));
    top = fmaxf(top, finite_abs(h[e]));
  }
  top = fmaxf(top, wave_xor(top, 16));
  top = fmaxf(top, wave_xor(top, 32));
  if (g == 0) part[wave][r] = top;
  lds_barrier();
#pragma unroll
  for (int q = 0; q < 8; ++q) top = fmaxf(top, part[q][r]);
  const int code = fp8_scale_code(top);
  if (m >= a.M) return;
  if (wave == 0 && g == 0) a.ys[m * a.ldys + fb] = (uint8_t)code;
  *(uint32_t*)((uint8_t*)a.y + m * a.ldy + n0) = fp8_scaled4(h[0], h[1], h[2], h[3], fp8_scale(code));
}

// ------------------------------------------------------------------------------------------------ host
template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED>
static void launch_tiles(Fp8Args a, hipStream_t s) {
  using C = Fp8Tile<TF, TM, WF, WM, NS, GATED>;
  a.m_tiles = (int)((a.M + C::BM - 1) / C::BM);
  a.f_tiles = (int)((a.N + C::OF - 1) / C::OF);
  const int64_t tiles = (int64_t)a.m_tiles * a.f_tiles;
  a.per_xcd = (int)((tiles + 7) / 8);
  // workgroups that fit a CU's LDS: two of 128 x 128 and 64 x 64 (73,728 and 77,824 bytes), one of the others (64 x 128: 83,968)
  constexpr int per_cu = std::min(4, 160 * 1024 / C::LDS);
  const int64_t wgs = std::min<int64_t>((int64_t)device_cu_count() / 8 * 8 * per_cu, 8 * (int64_t)a.per_xcd);
  fp8_tile_kernel<T, TF, TM, WF, WM, NS, GATED><<<dim3((unsigned)wgs), dim3(64 * C::NW), 0, s>>>(a);
}

// Checks shared by the products; rows: weight rows (N, or 2 N gated).  The stride of a single row means nothing: K stands for it
static int check_fp8(const char* what, Fp8Args& a, int64_t rows) {
  if (a.M < 0 || a.N < 1 || a.K < 16 || a.K % 16 || a.K > (1 << 22) || a.M > (1 << 30) || rows > (1 << 28))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: unsupported shape M=%lld N=%lld K=%d (K a multiple of 16 up to 2^22, M up to 2^30, "
                     "weight rows up to 2^28)", what, (long long)a.M, (long long)a.N, a.K);
  if (a.M == 0) return ATMA_OK;
  if (!a.x || !a.xs || !a.w || !a.ws || !a.y) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  if (a.M == 1) a.ldx = a.K;
  if (rows == 1) a.ldw = a.K;
  if ((uintptr_t)a.x % 16 || a.ldx % 16 || a.ldx < a.K || (uintptr_t)a.w % 16 || a.ldw % 16 || a.ldw < a.K)
    return set_error(ATMA_ERR_INVALID, "%s: rows of x and w must be 16-byte aligned and at least K long", what);
  if (a.ldxs < 0 || a.ldws < 0) return set_error(ATMA_ERR_INVALID, "%s: negative stride of scales", what);
  // a tile's rows (at most 256) are addressed by 32-bit byte offsets
  if (a.ldx > (1 << 23) || a.ldw > (1 << 23))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: rows more than 8 MiB apart", what);
  if (a.bias && (uintptr_t)a.bias % 4) return set_error(ATMA_ERR_INVALID, "%s: bias must be 4-byte aligned", what);
  if (a.bias && !dtype_size(a.bias_dtype))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: bias in fp32 or 16 bits (dtype %d)", what, a.bias_dtype);
  return ATMA_OK;
}

// What a tile shape costs: us a tile to begin and end it, and us a block of K, where few CUs work (latency) and where all do.
// Fitted to 30 shapes of 64 to 4,096 rows, 300 to 8,192 features and K 512 to 4,096, which it orders as measured but for
// differences under 10% (us: 1,000 x 1,024 -> 4,096 17.1 / 10.1 / 12.6 / 13.0 for 256 x 256, 128 x 128, 64 x 128 and 64 x 64,
// 4,000 x 512 -> 8,192 30 / 33 / 52 / 54, 64 x 4,096 -> 1,024 37 / 17.5 / 14.5 / 12.5; gated 777 x 1,024 -> 4,096 17.7 / 11.6 /
// 15.6 for 256, 128 and 64 tokens, 5,000 x 4,096 -> 1,024 47 / 60 / 59, 64 x 1,024 -> 4,096 15.0 / 9.6 / 8.2).
struct TileCost {
  int features, tokens;
  float tile, few, all;
};

static int cheapest(const Fp8Args& a, const TileCost* c, int n) {
  const float cus = (float)device_cu_count();
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < n; ++i) {
    const int64_t tiles = ((a.M + c[i].tokens - 1) / c[i].tokens) * ((a.N + c[i].features - 1) / c[i].features);
    const float fill = (float)tiles / cus;
    float t;
    if (fill <= 1.f) t = c[i].tile + (float)a.nk * (c[i].few + (c[i].all - c[i].few) * fill);
    else t = ceilf(fill) * (c[i].tile + (float)a.nk * c[i].all);
    if (i == 0 || t < least) best = i, least = t;
  }
  return best;
}

template <typename T, int MT, int FT, int NW = 4, int NS = 2>
static void launch_few(const Fp8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.N + 16 * FT - 1) / (16 * FT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  fp8_few_kernel<T, MT, FT, NW, NS><<<grid, dim3(64 * NW), 0, s>>>(a);
}

// The kernels of a product, in the order of the codes that atma_linear_fp8_form and atma_linear_gated_fp8_form return
enum LinearForm { kFew16x16, kFew32x16, kFew16x32, kFew32x32, kTile256x256, kTile128x128, kTile64x128, kTile64x64 };
enum GatedForm { kGatedFew, kGatedTile256, kGatedTile128, kGatedTile64 };

static int linear_form(const Fp8Args& a) {
  const int64_t cus = device_cu_count();
  // Few rows, while the split over K is what fills the card (us, split kernel / tiles, without bias; rows x K -> features).  Features in
  // sixteens up to a workgroup a CU, above it in two sixteens that share the tokens (64 x 1,024 -> 1,024 3.3 and 3.7, 32 x 1,024
  // -> 8,192 4.4 and 3.8), and no split past these borders: 64 x 4,096 -> 1,024 4.8 / 12.1, 64 x 1,024 -> 8,192 5.2 / 5.8, 256 x
  // 1,024 -> 4,096 8.8 / 6.1; 16 x 1,024 -> 24,576 5.3 / 6.7, 32 x 1,024 -> 24,576 7.3 / 6.9; weights that no L2 holds for the
  // second group of tokens, 64 x 8,192 -> 8,192, 27.2 / 21.5.
  const int64_t groups = (a.M + 31) / 32, narrow = groups * ((a.N + 15) / 16), wide = groups * ((a.N + 31) / 32);
  const int tokens = a.M <= 16 ? 16 : 32;
  if (narrow <= cus) return tokens == 16 ? kFew16x16 : kFew32x16;
  if (tokens == 16 && wide <= 3 * cus) return kFew16x32;
  if (a.M <= 32 ? 2 * wide <= 3 * cus : wide <= 2 * cus && a.N * a.K <= (32 << 20)) return kFew32x32;
  static constexpr TileCost kTiles[4] = {{256, 256, 5.5f, 1.15f, 1.72f},
                                         {128, 128, 1.2f, 0.50f, 0.72f},
                                         {64, 128, 1.3f, 0.36f, 0.42f},
                                         {64, 64, 0.7f, 0.32f, 0.30f}};
  return kTile256x256 + cheapest(a, kTiles, 4);
}

template <typename T>
static void launch_linear(const Fp8Args& a, hipStream_t s) {
  switch (linear_form(a)) {
    case kFew16x16: launch_few<T, 1, 1>(a, s); break;
    case kFew32x16: launch_few<T, 2, 1>(a, s); break;
    case kFew16x32: launch_few<T, 1, 2>(a, s); break;
    case kFew32x32: launch_few<T, 2, 2>(a, s); break;
    case kTile256x256: launch_tiles<T, 2, 4, 4, 2, 2, false>(a, s); break;
    case kTile128x128: launch_tiles<T, 2, 2, 2, 2, 2, false>(a, s); break;
    case kTile64x128: launch_tiles<T, 1, 2, 2, 2, 3, false>(a, s); break;
    default: launch_tiles<T, 1, 1, 2, 2, 4, false>(a, s); break;
  }
}

static int gated_form(const Fp8Args& a) {
  // Few rows: while a workgroup for every 16 tokens leaves none without a CU (us, split kernel / tiles; H 4,096, K 1,024: 128
  // rows 5.9 / 8.2, 256 rows, two a CU, 10.3 / 8.3; H 8,192, K 4,096, 64 rows 15.7 / 20.2) and LDS holds their K
  const int64_t blocks = a.N / kFp8Block, groups = (a.M + 15) / 16;
  if (blocks * groups <= device_cu_count() && a.nk <= kGatedFewBlocks) return kGatedFew;
  static constexpr TileCost kTiles[3] = {{128, 256, 5.0f, 1.00f, 1.60f},
                                         {128, 128, 1.7f, 0.70f, 0.98f},
                                         {128, 64, 1.3f, 0.53f, 0.63f}};
  return kGatedTile256 + cheapest(a, kTiles, 3);
}

static void launch_gated(const Fp8Args& a, hipStream_t s) {
  switch (gated_form(a)) {
    case kGatedFew:
      fp8_gated_few_kernel<<<dim3((unsigned)(a.N / kFp8Block), (unsigned)((a.M + 15) / 16)), dim3(512), 0, s>>>(a);
      break;
    case kGatedTile256: launch_tiles<bf16, 2, 4, 4, 2, 2, true>(a, s); break;
    case kGatedTile128: launch_tiles<bf16, 2, 2, 4, 2, 2, true>(a, s); break;
    default: launch_tiles<bf16, 2, 1, 4, 2, 3, true>(a, s); break;
  }
}

// A product's sizes alone, within the limits of check_fp8; K 0 where they are not
static Fp8Args fp8_sizes(int64_t M, int64_t N, int64_t K) {
  Fp8Args a{};
  if (M < 1 || N < 1 || K < 16 || K % 16 || K > (1 << 22) || M > (1 << 30) || N > (1 << 28)) return a;
  a.M = M;
  a.N = N;
  a.K = (int)K;
  a.nk = (int)((K + kFp8Block - 1) / kFp8Block);
  return a;
}

}  // namespace atma

extern "C" int atma_linear_fp8(const void* x, int64_t ldx, const void* xs, int64_t ldxs, const void* w, int64_t ldw,
                               const void* ws, int64_t ldws, const void* bias, int bias_dtype, void* y, int64_t ldy,
                               int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  using namespace atma;
  if (dtype != ATMA_BF16 && dtype != ATMA_F16)
    return set_error(ATMA_ERR_UNSUPPORTED, "linear_fp8: 16-bit output only (dtype %d)", dtype);
  if (K < 0 || K > (1 << 22)) return set_error(ATMA_ERR_UNSUPPORTED, "linear_fp8: K=%lld", (long long)K);
  Fp8Args a{(const uint8_t*)x, ldx, (const uint8_t*)xs, ldxs, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws,
            (N + kFp8Block - 1) / kFp8Block, bias, bias_dtype, y, ldy, nullptr, 0, M, N, (int)K, (int)((K + kFp8Block - 1) / kFp8Block), 0, 0, 0};
  if (const int rc = check_fp8("linear_fp8", a, N)) return rc;
  if (M == 0) return ATMA_OK;
  if (ldy < N || (uintptr_t)y % 2)
    return set_error(ATMA_ERR_INVALID, "linear_fp8: rows of y must be at least N long, at an address of their type");
  if (dtype == ATMA_BF16) launch_linear<bf16>(a, (hipStream_t)stream);
  else launch_linear<f16>(a, (hipStream_t)stream);
  return check_launch("linear_fp8");
}

extern "C" int atma_linear_gated_fp8(const void* x, int64_t ldx, const void* xs, int64_t ldxs, const void* w,
                                     int64_t ldw, const void* ws, int64_t ldws, const void* bias, int bias_dtype,
                                     void* y, int64_t ldy, void* ys, int64_t ldys, int64_t M, int64_t H, int64_t K,
                                     void* stream) {
  using namespace atma;
  if (K < 0 || K > (1 << 22)) return set_error(ATMA_ERR_UNSUPPORTED, "linear_gated_fp8: K=%lld", (long long)K);
  Fp8Args a{(const uint8_t*)x, ldx, (const uint8_t*)xs, ldxs, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws,
            2 * H / kFp8Block, bias, bias_dtype, y, ldy, (uint8_t*)ys, ldys, M, H, (int)K, (int)((K + kFp8Block - 1) / kFp8Block), 0, 0, 0};
  if (H < kFp8Block || H % kFp8Block || H > (1 << 27))
    return set_error(ATMA_ERR_UNSUPPORTED, "linear_gated_fp8: H must be a multiple of %d (got %lld)", kFp8Block,
                     (long long)H);
  if (const int rc = check_fp8("linear_gated_fp8", a, 2 * H)) return rc;
  if (M == 0) return ATMA_OK;
  if (!ys || (uintptr_t)y % 16 || ldy % 16 || ldy < H || ldys < H / kFp8Block)
    return set_error(ATMA_ERR_INVALID, "linear_gated_fp8: rows of y must be 16-byte aligned and at least H long");
  launch_gated(a, (hipStream_t)stream);
  return check_launch("linear_gated_fp8");
}

extern "C" int atma_linear_fp8_form(int64_t M, int64_t N, int64_t K) {
  const atma::Fp8Args a = atma::fp8_sizes(M, N, K);
  return a.K ? atma::linear_form(a) : -1;
}

extern "C" int atma_linear_gated_fp8_form(int64_t M, int64_t H, int64_t K) {
  const atma::Fp8Args a = atma::fp8_sizes(M, H, K);
  return a.K && H % atma::kFp8Block == 0 && H <= (1 << 27) ? atma::gated_form(a) : -1;
}
