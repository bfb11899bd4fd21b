// Products with 4-bit weights: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]) for 16-bit x (M, K) and w (N, K) in the format of
// fp4.h, and the MLP's first projection with its activation, gate * relu(a)^2 of the fp32 sums.  No reference counterpart.
//
// The weights become the matrix instructions' 16-bit operands in registers, one instruction for two of them, scale included
// (fp4_unpack8), so what is read from memory and LDS for them stays at 4.25 bits.  The order of k within an instruction is
// free as long as both operands follow it: a lane takes 16 bytes of a weight row, one group of 32 with its one scale, and the
// same 32 k of a token, four 16-byte pieces.
#include <algorithm>

#include "fp4.h"
#include "gemm_tiles.h"

namespace atma {

constexpr int kFp4Block = 64;  // of K, a stage of the tiles' ring: 128 bytes of a token's row, 32 of a weight's

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
  int K, nk;  // nk: blocks of K
  int m_tiles, f_tiles, per_xcd;
};

template <typename T>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  Pack8 pa, pb;
  pa.u = a;
  pb.u = b;
  if constexpr (__is_same(T, bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa.b, pb.b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(pa.h, pb.h, c, 0, 0, 0);
}

// The kernel's arguments read again where they are needed: kept in scalar registers through the loop they would be spilled
typedef const __attribute__((address_space(4))) Fp4Args* LateArgs4;
__device__ __forceinline__ LateArgs4 late_args4() {
  LateArgs4 p = (LateArgs4)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// ------------------------------------------------------------------------------------------------ tiles
// A workgroup of WF x WM waves owns BF weight rows x BM tokens, a wave TF x TM tiles of 32 x 32.  K runs in blocks of 64 through a
// ring of NS stages in LDS, filled by direct copies.  A block is four steps of 16 k a lane half: while the products of a
// step run from registers, the operands of the next one are read into a second set, the weights converted.  Before the last step
// the waves meet: the next block has landed, this one's stage is free, and the copies of block k + NS go there over the next
// four steps.  The workgroup is persistent and all of this runs on across its tiles: a tile's first copies fly and its
// first operands are read during the last blocks of the one before.
//
// A block of 256 x 256 takes 2,760 cycles, 2,048 of them products: two waves share a SIMD, and while one runs its steps
// at 1.1 to 1.3 times the time of their products, what both lose lies behind the barrier.  Measured without gain: products ahead
// of the reads in each step, a higher priority for the products, the weights' conversion behind the last step's products,
// 128 x 64 tiles a wave instead of 64 x 128 (twice the conversions, two thirds of the reads), operands read a whole block ahead.
// 65,536 x 4,096 -> 1,024 takes 430 to 458 us by the card (1.2 PFLOP/s, matrix cores busy 70 % at the 1.7 GHz that power allows), the
// library's 16-bit product on weights already converted 356 to 376, converted in the call 368 to 370.
// Small tiles, a wave a SIMD, are bound by issue: a block of 128 x 32 is 130 instructions and 128 cycles of products in 700.
//
// The weights are the MFMA's rows, in an order such that a lane's accumulators are 16 consecutive features of one token
// (row 8 q + 4 h + e is feature 16 h + 4 q + e).  Their rows are 32 bytes in LDS, chunk c of row r at position
// c ^ (r / 16) % 2: the 16 lanes that read one chunk of 16 such rows cover all banks.
//
// KS = 2: two such sets of waves, each with a ring of its own, take half of K each, and the first adds the second's sums, which come
// through LDS.  For tiles that are few: their time is the chain of blocks, and two waves a SIMD issue beside each other.
template <int TF, int TM, int WF, int WM, int NS_, bool GATED, int KS = 1>
struct Fp4Tile {
  static constexpr int NW = WF * WM, NS = NS_;
  static constexpr int BF = 32 * TF * WF, BM = 32 * TM * WM;
  static constexpr int OF = GATED ? BF / 2 : BF;  // output features
  static constexpr int TO = GATED ? TF / 2 : TF;  // tiles of output features a wave
  static constexpr int W = BM * 128, STAGE = W + BF * 32;
  static constexpr int COPIES = 2 + BM / 8 / NW;  // a wave and block: scales, 32 weight rows, 8 token rows each
  static constexpr int FIRST = COPIES / 4;        // of them in the last step of a block
  static constexpr int RING = NS + 2;    // blocks and tiles under way: copies run NS blocks ahead
  static constexpr int SLOT = NW * 256;  // a block's scales, in words: two a weight row
  static constexpr int AUX = NS * STAGE, BIAS = AUX + RING * SLOT, TURN = BIAS + RING * 1024, SET = TURN + 2048 * NW;
  static constexpr int JOIN = KS * SET, LDS = JOIN + (KS - 1) * NW * TF * TM * 4096;
  static_assert(BF == 32 * NW && BM % (8 * NW) == 0 && BF <= 256 && NW > 2, "whole copies, a bias of 1 KiB, copied by wave 2");
  static_assert(!GATED || TF % 2 == 0, "a gated wave has its features' a and gate rows");
  static_assert(NS >= 3 && (NS - 1) * COPIES < 63, "vmcnt counts to 63");
};

template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED, int KS>
__global__ void __launch_bounds__(64 * WF * WM * KS, 2) fp4_tile_kernel(Fp4Args a) {
  using C = Fp4Tile<TF, TM, WF, WM, NS, GATED, KS>;
  constexpr int TO = C::TO;
  __shared__ __attribute__((aligned(1024))) uint8_t all_lds[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int any_wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int set = KS == 1 ? 0 : any_wave / C::NW, wave = any_wave - set * C::NW;
  uint8_t* lds = all_lds + set * C::SET;
  const int wf = wave % WF, wm = wave / WF;
  const int r = lane & 31, h = lane >> 5;
  const int nk = (a.nk + KS - 1) / KS, pk0 = set * nk;  // the set's blocks of K
  int64_t m0, f0;
  int u = blockIdx.x >> 3;
  if (!gemm_tile_at<C>(a, blockIdx.x & 7, u, m0, f0)) return;

  // ---- the copies, NS blocks ahead.  Token copy i of a wave moves rows 8 (i NW + wave) .. + 7, lane l the chunk that belongs
  // at position l % 8 of row l / 8; the weights' copy rows 32 wave .. + 31, lane l the chunk of position l % 2 of row l / 2;
  // the scales' copy the same rows' codes, lane l group l % 2 of row l / 2.  Out of range (chunks past K, rows past the
  // end, everything behind the last tile) zeros are written; scales past K or the last row are the last ones
  const uint32_t lds0 = lds_offset(lds);
  const int crow = 8 * wave + (lane >> 3);
  const int xk = 16 * ((lane & 7) ^ x_swizzle(crow));  // bytes into the row
  const uint32_t xv0 = (uint32_t)crow * (uint32_t)(2 * a.ldx) + (uint32_t)xk, xstep = 8u * C::NW * (uint32_t)(2 * a.ldx);
  const int wk = 16 * ((lane & 1) ^ (lane >> 5));
  constexpr int half = C::NW / 2;  // gated: the first half of the waves copy a rows, the others gate rows
  const int wbase = 32 * (GATED ? wave % half : wave);
  const uint32_t wv0 = (uint32_t)(wbase + (lane >> 1)) * (uint32_t)a.ldw + (uint32_t)wk;
  __amdgpu_buffer_rsrc_t xr, wr;
  const uint8_t* scales;  // the first code of a lane's weight row
  int pu = u, pk = pk0, plimit = 0, ptile = 0, pslot = 0, pstage = 0;
  auto aim = [&](int64_t tm0, int64_t tf0) {
    LateArgs4 p = late_args4();
    const int64_t rows = min((int64_t)C::BM, p->M - tm0);
    xr = buffer_rsrc((const uint16_t*)p->x + tm0 * p->ldx, (uint32_t)(rows * 2 * p->ldx));
    const int64_t n0 = GATED && wave >= half ? p->N + tf0 : tf0;
    wr = buffer_rsrc(p->w + n0 * p->ldw, (uint32_t)(min((int64_t)C::OF, p->N - tf0) * p->ldw));
    const int64_t last = (GATED && wave >= half ? 2 : 1) * p->N - 1;
    scales = p->ws + min(n0 + wbase + (lane >> 1), last) * p->ldws;
    plimit = p->K;
    if (p->bias && wave == 2 && set == 0) {
      // the tile's biases (gated: those of a, then of gate), a word each, to its slot
      const bool wide = p->bias_dtype == ATMA_F32;
      for (int i = 0; i < C::BF / 64; ++i) {
        const int f = 64 * i + lane;
        const int64_t n = min(GATED && f >= C::OF ? p->N + tf0 + f - C::OF : tf0 + f, (GATED ? 2 : 1) * p->N - 1);
        const uint32_t at = lds0 + C::BIAS + 1024 * ptile + 256 * i;
        if (wide) dma_load4_at((const uint32_t*)p->bias + n, at);
        else dma_load2_at((const uint16_t*)p->bias + n, at);
      }
    }
    ptile = ptile + 1 == C::RING ? 0 : ptile + 1;
  };
  auto next_tile = [&]() {
    int64_t nm0, nf0;
    pk = pk0;
    pu += gridDim.x >> 3;
    if (gemm_tile_at<C>(*late_args4(), blockIdx.x & 7, pu, nm0, nf0)) aim(nm0, nf0);
    else plimit = 0;
  };
  uint32_t pd, pxv, pwv;
  uint32_t ps;
  const uint8_t* pscale;
  auto copies_begin = [&]() {
    if (pk == pk0 + nk) next_tile();
    pscale = scales + max(0, min(2 * pk + (lane & 1), plimit / kFp4Group - 1));
    ps = lds0 + C::AUX + C::SLOT * pslot + 256 * wave;
    pslot = pslot + 1 == C::RING ? 0 : pslot + 1;
    pd = lds0 + pstage * C::STAGE + 1024 * wave;
    pstage = pstage + 1 == NS ? 0 : pstage + 1;
    const int k = kFp4Block * pk++;
    pxv = k + xk / 2 < plimit ? xv0 + 2u * (uint32_t)k : 0x80000000u;
    pwv = k + 2 * wk < plimit ? wv0 + (uint32_t)k / 2 : 0x80000000u;
  };
  auto copy = [&](int i) {
    if (i == 0) dma_load1_at(pscale, ps);
    else if (i == 1) dma_buf16_at(wr, pwv, 0u, pd + C::W);
    else dma_buf16_at(xr, pxv + (i - 2) * xstep, 0u, pd + 1024 * C::NW * (i - 2));
  };

  // ---- operand reads
  const int wrow0 = 32 * TO * wf;  // the wave's first output feature in the tile
  const int wrow = 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
  auto wtile = [](int t) { return GATED ? t / TO * (C::BF / 2) + 32 * (t % TO) : 32 * t; };
  const uint32_t wofs = (uint32_t)(C::W + (wrow0 + wrow) * 32 + 16 * (h ^ ((r >> 2) & 1)));
  const uint32_t sofs = (uint32_t)(C::AUX + 8 * (wrow0 + wrow) + 4 * h);
  uint32_t xofs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) xofs[j] = (uint32_t)((32 * TM * wm + r) * 128 + 16 * ((4 * h + j) ^ x_swizzle(r)));
  f32x16 acc[TF][TM];
  u32x4 raw[TF], wv[2][TF], xv[2][TM];
  uint32_t code[TF];
  int stage = 0, slot = 0, tile = 0;  // what is read next
  auto read_w = [&](const uint8_t* base, int t) {
    raw[t] = *(const u32x4*)(base + wofs + 32 * wtile(t));
    code[t] = *(const uint32_t*)(lds + sofs + C::SLOT * slot + 8 * wtile(t));
  };
  auto convert = [&](int s, int j, int t) {
    wv[s][t] = fp4_unpack8<T>(raw[t][j], __builtin_bit_cast(float, code[t] << 23));
    asm volatile("" : "+v"(wv[s][t]));  // here, not where it is used
  };
  auto read_x = [&](const uint8_t* base, int j, int t) { xv[j & 1][t] = *(const u32x4*)(base + xofs[j] + 4096 * t); };

  aim(m0, f0);
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) {
    copies_begin();
#pragma unroll
    for (int c = 0; c < C::COPIES; ++c) copy(c);
  }
  copies_begin();
#pragma unroll
  for (int c = 0; c < C::FIRST; ++c) copy(c);
  wait_vmcnt<(NS - 2) * C::COPIES + C::FIRST>();
  lds_barrier();
#pragma unroll
  for (int t = 0; t < TF; ++t) read_w(lds, t);
#pragma unroll
  for (int t = 0; t < TM; ++t) read_x(lds, 0, t);
#pragma unroll
  for (int t = 0; t < TF; ++t) convert(0, 0, t);
  slot = 1;
  while (true) {
    // ---- the sums start from the bias
#pragma unroll
    for (int t = 0; t < TF; ++t) {
      float b[16] = {};
      const int f = wrow0 + 16 * h + (GATED ? t / TO * C::OF + 32 * (t % TO) : 32 * t);
      LateArgs4 p = late_args4();
      if (p->bias && set == 0) {
        const uint8_t* at = lds + C::BIAS + 1024 * tile;
        const int dtype = p->bias_dtype;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const u32x4 v = *(const u32x4*)(at + 4 * (f + e));
#pragma unroll
          for (int i = 0; i < 4; ++i) b[e + i] = bias_f32(dtype, v[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][j][e] = b[e];
    }
    tile = tile + 1 == C::RING ? 0 : tile + 1;

    for (int kb = 0; kb < nk; ++kb) {
      const uint8_t* base = lds + stage * C::STAGE;
      stage = stage + 1 == NS ? 0 : stage + 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j == 3) {
          // the next block's copies have landed in every wave, and every wave has read this block
          wait_vmcnt<(NS - 2) * C::COPIES>();
          lds_barrier();
          base = lds + stage * C::STAGE;
        }
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          __builtin_amdgcn_sched_barrier(0);
          // ahead of the products of token tile m: a share of the next step's operands, all of them in the first half of the step
          if (j == 3 && m == 0) {
#pragma unroll
            for (int t = 0; t < TF; ++t) read_w(base, t);
            slot = slot + 1 == C::RING ? 0 : slot + 1;
          }
#pragma unroll
          for (int t = 2 * m; t < min(2 * m + 2, TM); ++t) read_x(base, (j + 1) & 3, t);
#pragma unroll
          for (int t = 0; t < TF; ++t) acc[t][m] = mfma32<T>(wv[j & 1][t], xv[j & 1][m], acc[t][m]);
          const int q = (j + 1) & 3, c0 = q * C::COPIES / 4, c1 = (q + 1) * C::COPIES / 4;  // this step's copies
#pragma unroll
          for (int c = c0 + m * (c1 - c0) / TM; c < c0 + (m + 1) * (c1 - c0) / TM; ++c) copy(c);
          // (the last step's first half waits for the next block's weights)
          const int from = j == 3 ? max(0, 2 * m - TM) : m, share = j == 3 && TM > 1 ? 2 : 1;
          if (j != 3 || TM == 1 || 2 * m >= TM) {
#pragma unroll
            for (int t = 0; t < TF; ++t)
              if (t >= from * TF / TM && t < (from + share) * TF / TM) convert((j + 1) & 1, (j + 1) & 3, t);
          }
        }
        if (j == 2) copies_begin();  // (the addresses: nothing keeps the products behind the barrier waiting)
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- epilogue of tile (m0, f0): token 32 (TM wm + j) + r, 16 consecutive features a tile.  Through LDS, a wave its own 2 KiB:
    // 32 tokens x 32 features at a time turn from a token a lane to 64-byte pieces, four lanes each (chunk c of row r at position
    // c ^ (r / 4) % 4)
    if constexpr (KS > 1) {
      // (the buffer is written again behind the barriers of the next tile's blocks)
      f32x4* join = (f32x4*)(all_lds + C::JOIN) + wave * TF * TM * 256 + lane;
      if (set) {
#pragma unroll
        for (int i = 0; i < TF * TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const f32x16& v = acc[i / TM][i % TM];
            join[256 * i + 16 * e] = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
          }
      }
      lds_barrier();
      if (!set) {
#pragma unroll
        for (int i = 0; i < TF * TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const f32x4 v = join[256 * i + 16 * e];
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i / TM][i % TM][e + q] += v[q];
          }
      }
    }
    LateArgs4 p = late_args4();
    const bool whole = f0 + C::OF <= p->N;  // every feature of the tile
    uint8_t* turn = lds + C::TURN + 2048 * wave;
    const int64_t ldy = p->ldy, N = p->N, M = p->M;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      if (set) break;
#pragma unroll
      for (int t = 0; t < TO; ++t) {
        f32x16 v = acc[t][j];
        if constexpr (GATED) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = gate_act(v[e], acc[TO + t][j][e]);
        }
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
    u += gridDim.x >> 3;
    if (!gemm_tile_at<C>(*late_args4(), blockIdx.x & 7, u, m0, f0)) break;
  }
  wait_vmcnt<0>();  // no copy outlives its workgroup's LDS
}

__device__ __forceinline__ float fp4_bias(const Fp4Args& a, int64_t n) {
  if (!a.bias) return 0.f;
  return bias_f32(a.bias_dtype, a.bias_dtype == ATMA_F32 ? ((const uint32_t*)a.bias)[n] : ((const uint16_t*)a.bias)[n]);
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 MT tokens at a time: latency and the stream of weights.  A wave owns FT tiles of 16 features (gated: 16 a rows and the
// gate rows of the same features), or one of `splits` shares of their K, whose sums are joined through LDS in a fixed order.
// It has a ring of its own of NS blocks of 256 k, filled by direct copies of whole 128-byte lines of the weights, and waits
// for nothing but its own copies.  The tokens lie in LDS, all of K, copied once (RING: where they do not fit, a
// block of them comes with each block of weights).  A workgroup walks over its tiles, and the ring runs on across them.
//
// Its time is latency, launch, first copies, join: 1 x 4,096 -> 1,024 5.1 us (2.2 MB), 16 x 1,024 -> 4,096 4.5, gated 5.3; 1 x 1,024 -> 50,304
// streams 27 MB in 8.2.  Four waves with a ring for the tokens too beat eight with the tokens kept wherever the ring's copies of the tokens
// (8 KiB a block of 2 KiB of weights, from L2) are few: see choose_fp4.
//
// v_mfma_f32_16x16x32: lane (r, g) takes chunks g and g + 4 of a weight row's eight, one group of 32 k each with its scale, and
// the same k of token r.  Chunk c of a weight row lies at position c ^ (r / 2) % 8, chunk c of a token's row at c ^ r % 16.
constexpr int kFewBlock = 256;
constexpr int kFewTokens = 64 * 1024;  // LDS for the tokens

struct Fp4FewArgs {
  Fp4Args a;
  int tiles, log_splits;  // tiles of 16 FT weight rows (gated: of 16 features); splits of K, a power of two up to the blocks of K
};

template <int MT, int FT, int NW, bool RING>
struct Fp4Few {
  static constexpr int NS = RING ? 2 : 4;
  static constexpr int WCOPY = 2 * FT, XCOPY = RING ? 8 * MT : 0, COPIES = 2 * WCOPY + XCOPY;
  static constexpr int X = FT * (2048 + 512), STAGE = X + 1024 * XCOPY;
  static constexpr int TOKENS = NW * NS * STAGE, RED = TOKENS + (RING ? 0 : kFewTokens), LDS = RED + NW * FT * MT * 1024;
};

template <typename T, int MT, int FT, int NW, bool RING, bool GATED>
__global__ void __launch_bounds__(64 * NW) fp4_few_kernel(Fp4FewArgs f) {
  using C = Fp4Few<MT, FT, NW, RING>;
  constexpr int NS = C::NS, OT = GATED ? 1 : FT;  // tiles of output features
  const Fp4Args& a = f.a;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int ls = f.log_splits, splits = 1 << ls, share = wave & (splits - 1), nk = a.nk;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * MT;
  const int rows = (int)min((int64_t)16 * MT, a.M - m0);
  const __amdgpu_buffer_rsrc_t xr = buffer_rsrc((const uint16_t*)a.x + m0 * a.ldx, (uint32_t)(rows * 2 * a.ldx));
  const uint32_t ring0 = lds_offset(lds) + wave * NS * C::STAGE;
  auto tile_of = [&](int it) { return ((it << (31 - __builtin_clz(NW) - ls)) + (wave >> ls)) * (int)gridDim.x + (int)blockIdx.x; };

  // ---- the weights' copies.  Copy i of a block moves rows 8 i .. + 7, lane l the chunk that belongs at position l % 8 of row
  // l / 8; the scales' copies the same rows' codes, lane l group l % 8.  Chunks past K, rows past the end and tiles past the last
  // one are zeros, scales there the nearest ones
  const int crow = lane >> 3;
  __amdgpu_buffer_rsrc_t wr[2];
  const uint8_t* codes[2 * FT];
  int pit = 0, pkb = share, plimit = 0;
  auto aim = [&]() {
    const int tile = tile_of(pit);
    plimit = tile < f.tiles ? a.K : 0;
    const int64_t n0 = min((int64_t)tile * 16 * OT, a.N - 1);
    wr[0] = buffer_rsrc(a.w + n0 * a.ldw, (uint32_t)(min((int64_t)16 * OT, a.N - n0) * a.ldw));
    if constexpr (GATED) wr[1] = buffer_rsrc(a.w + (a.N + n0) * a.ldw, (uint32_t)(min((int64_t)16, a.N - n0) * a.ldw));
#pragma unroll
    for (int i = 0; i < 2 * FT; ++i) {
      const int64_t n = GATED && i >= 2 ? a.N + min(n0 + 8 * (i - 2) + crow, a.N - 1) : min(n0 + 8 * i + crow, a.N - 1);
      codes[i] = a.ws + n * a.ldws;
    }
  };
  auto copies = [&](int slot) {
    const uint32_t d = ring0 + slot * C::STAGE;
    const int k0 = kFewBlock * pkb, group = min(8 * pkb + (lane & 7), a.K / kFp4Group - 1);
#pragma unroll
    for (int i = 0; i < 2 * FT; ++i) {
      const int row = 8 * i + crow, at = GATED ? row & 15 : row;
      const int chunk = (lane & 7) ^ x_swizzle(row);
      const uint32_t v = (uint32_t)at * (uint32_t)a.ldw + 128u * (uint32_t)pkb + 16u * (uint32_t)chunk;
      dma_buf16_at(wr[GATED ? i / 2 : 0], k0 + 32 * chunk < plimit ? v : 0x80000000u, 0u, d + 1024 * i);
    }
#pragma unroll
    for (int i = 0; i < 2 * FT; ++i) dma_load1_at(codes[i] + group, d + FT * 2048 + 256 * i);
    if constexpr (RING) {
      // two token rows of 512 bytes a copy
#pragma unroll
      for (int i = 0; i < C::XCOPY; ++i) {
        const int row = 2 * i + (lane >> 5), chunk = (lane & 31) ^ (row & 15);
        const uint32_t v = (uint32_t)row * (uint32_t)(2 * a.ldx) + 512u * (uint32_t)pkb + 16u * (uint32_t)chunk;
        dma_buf16_at(xr, k0 + 8 * chunk < plimit ? v : 0x80000000u, 0u, d + C::X + 1024 * i);
      }
    }
    pkb += splits;
    if (pkb >= nk) {
      pkb = share;
      ++pit;
      aim();
    }
  };
  if constexpr (!RING) {
    // chunk i of the tokens' rows, 32 nk chunks each
    const int per = 32 * nk, total = rows * per;
    for (int i0 = 64 * wave; i0 < total; i0 += 64 * NW) {
      const int i = i0 + lane, row = i / per, at = i - row * per, chunk = at ^ (row & 15);
      dma_buf16_at(xr, row < rows && 8 * chunk < a.K ? (uint32_t)row * (uint32_t)(2 * a.ldx) + 16u * (uint32_t)chunk : 0x80000000u,
                   0u, lds_offset(lds) + C::TOKENS + 16 * i0);
    }
  }
  aim();
#pragma unroll
  for (int i = 0; i < NS; ++i) copies(i);
  if constexpr (!RING) {
    wait_vmcnt<NS * C::COPIES>();
    lds_barrier();  // the tokens are there, from every wave
  }

  int slot = 0;
  for (int it = 0;; ++it) {
    const int tile = tile_of(it);
    if (splits == 1 ? tile >= f.tiles : tile_of(it) - (wave >> ls) * (int)gridDim.x >= f.tiles) break;  // (the same for every wave that joins)
    const int64_t n0 = (int64_t)tile * 16 * OT + 4 * g;
    f32x4 acc[FT][MT] = {};
    for (int kb = share; kb < nk; kb += splits) {
      wait_vmcnt<(NS - 1) * C::COPIES>();
      const uint8_t* base = lds + wave * NS * C::STAGE + slot * C::STAGE;
      u32x4 raw[2][FT], xv[2][MT][4];
      uint32_t code[2][FT];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int t = 0; t < FT; ++t) {
          raw[q][t] = *(const u32x4*)(base + 2048 * t + 128 * r + 16 * ((4 * q + g) ^ x_swizzle(r)));
          code[q][t] = *(const uint32_t*)(base + FT * 2048 + 512 * t + 32 * r + 4 * (4 * q + g));
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int row = RING ? 16 * j + r : min(16 * j + r, rows - 1);
          const uint8_t* xp = RING ? base + C::X + 512 * row : lds + C::TOKENS + 512 * (row * nk + kb);
#pragma unroll
          for (int e = 0; e < 4; ++e) xv[q][j][e] = *(const u32x4*)(xp + 16 * ((16 * q + 4 * g + e) ^ (row & 15)));
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the copies that overwrite them start
      copies(slot);
      slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int t = 0; t < FT; ++t) {
          const float scale = __builtin_bit_cast(float, code[q][t] << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u32x4 wv = fp4_unpack8<T>(raw[q][t][e], scale);
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[t][j] = mfma16x16x32<T>(wv, xv[q][j][e], acc[t][j]);
          }
        }
    }
    if (splits > 1) {
      auto red = (f32x4(*)[FT][MT][64])(lds + C::RED);
#pragma unroll
      for (int t = 0; t < FT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) red[wave][t][j][lane] = acc[t][j];
      lds_barrier();
    }
    // every share stores some of the outputs
#pragma unroll
    for (int o = 0; o < OT * MT; ++o) {
      if ((o & (splits - 1)) != share) continue;
      const int t = o / MT, j = o % MT;
      f32x4 v = acc[t][j], gate = acc[FT - 1][j];
      if (splits > 1) {
        auto red = (const f32x4(*)[FT][MT][64])(lds + C::RED);
        const int first = wave & ~(splits - 1);
        v = red[first][t][j][lane];
        gate = red[first][FT - 1][j][lane];
        for (int q = 1; q < splits; ++q) {
          v += red[first + q][t][j][lane];
          if constexpr (GATED) gate += red[first + q][FT - 1][j][lane];
        }
      }
      const int64_t m = m0 + 16 * j + r, n = n0 + 16 * t;
      if (16 * j + r >= rows || n >= a.N) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t ne = min(n + e, a.N - 1);
        v[e] += fp4_bias(a, ne);
        if constexpr (GATED) v[e] = gate_act(v[e], gate[e] + fp4_bias(a, a.N + ne));
      }
      T* y = (T*)a.y + m * a.ldy + n;
      if (n + 4 <= a.N) {
        *(u32x2_any*)y = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.N) y[e] = from_f32<T>(v[e]);
      }
    }
    if (splits > 1) lds_barrier();  // the sums are read before the next tile's are written
  }
  wait_vmcnt<0>();  // no copy outlives its workgroup's LDS
}

template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED, int KS = 1>
static void launch_tiles4(Fp4Args a, hipStream_t s) {
  using C = Fp4Tile<TF, TM, WF, WM, NS, GATED, KS>;
  a.m_tiles = (int)((a.M + C::BM - 1) / C::BM);
  a.f_tiles = (int)((a.N + C::OF - 1) / C::OF);
  const int64_t tiles = (int64_t)a.m_tiles * a.f_tiles;
  a.per_xcd = (int)((tiles + 7) / 8);
  constexpr int per_cu = 160 * 1024 / C::LDS;
  const int64_t wgs = std::min<int64_t>((int64_t)device_cu_count() / 8 * 8 * per_cu, 8 * (int64_t)a.per_xcd);
  fp4_tile_kernel<T, TF, TM, WF, WM, NS, GATED, KS><<<dim3((unsigned)wgs), dim3(64 * C::NW * KS), 0, s>>>(a);
}

// How the few rows' kernel is laid over the card
struct FewPlan {
  int tiles, groups, log_splits, wgs, steps;  // steps: the blocks of K that a wave goes through
};

template <int MT, int FT, int NW, bool RING, bool GATED>
static FewPlan plan_few4(const Fp4Args& a) {
  using C = Fp4Few<MT, FT, NW, RING>;
  constexpr int OF = 16 * (GATED ? 1 : FT);
  FewPlan p{(int)((a.N + OF - 1) / OF), (int)((a.M + 16 * MT - 1) / (16 * MT)), 0, 0, 0};
  const int cus = device_cu_count(), nk = (a.K + kFewBlock - 1) / kFewBlock;
  // K is split among a workgroup's waves while every workgroup still finds a CU
  while ((2 << p.log_splits) <= std::min(NW, nk) && (int64_t)p.tiles * p.groups * (2 << p.log_splits) <= (int64_t)cus * NW)
    ++p.log_splits;
  const int at_once = NW >> p.log_splits;  // tiles of a workgroup
  p.wgs = std::min((p.tiles + at_once - 1) / at_once, std::max(1, cus * (160 * 1024 / C::LDS) / p.groups));
  p.steps = (p.tiles + at_once * p.wgs - 1) / (at_once * p.wgs) * ((nk + (1 << p.log_splits) - 1) >> p.log_splits);
  return p;
}

template <typename T, int MT, int FT, int NW, bool RING, bool GATED>
static void launch_few4(const Fp4Args& a, hipStream_t s) {
  const FewPlan p = plan_few4<MT, FT, NW, RING, GATED>(a);
  Fp4FewArgs f{a, p.tiles, p.log_splits};
  f.a.nk = (a.K + kFewBlock - 1) / kFewBlock;
  fp4_few_kernel<T, MT, FT, NW, RING, GATED><<<dim3((unsigned)p.wgs, (unsigned)p.groups), dim3(64 * NW), 0, s>>>(f);
}

// The kernel for a product: the one with the least time by a cost of its form, us of a graph's launch.  The few rows' kernel:
// a part that does not depend on the size, the steps of a wave, and all blocks of all waves over the card's SIMDs.  The tiles:
// TileCost and a part that does not depend on the size.  Fitted to 221 measured shapes of 1 to 16,384 rows, 512 to 50,304 features and K
// of 256 to 4,096: over them the choice takes 1.0 % longer than the best of all forms in the mean and 15 % at most (gated: 0.6 % and
// 12 %).  What each form is there for (us, it and the best of the others):
//   16 rows a workgroup through a ring    16 x 4,096 -> 1,024     5.8 and  7.5    128 x 1,024 -> 1,024    4.9 and  5.3
//   32 rows a workgroup through a ring   192 x 4,096 -> 1,024    11.0 and 13.2     32 x 4,096 -> 8,192   10.6 and 12.6
//   16 rows' K kept in LDS                 1 x 1,024 -> 50,304    8.2 and 14.2      8 x 4,096 -> 8,192    7.0 and  8.0
//   tiles of 128 features x 32 tokens     32 x 1,024 -> 50,304   10.4 and 12.0
//   tiles of 128 x 64                     64 x 1,024 -> 50,304   13.1 and 16.3
//   tiles of 128 x 128                   512 x 4,096 -> 8,192    39.1 and 50.7
//   tiles of 256 x 256                16,384 x 4,096 -> 1,024   107   and 135
//   tiles of 128 x 32, K in halves       512 x 4,096 -> 1,024    16.8 and 18.8    777 x 1,024 -> 1,024    7.2 and  8.1
//   tiles of 128 x 64, K in halves       192 x 4,096 -> 8,192    21.9 and 27.1    512 x 1,024 -> 4,096    8.8 and  9.9
// gated: 64 x 64 with K in halves for 256 x 1,024 -> 4,096 9.3 and 11.5 (all K 10.2), 64 x 128 for 512 12.8 and 16.6, 128 x 256 for 8,192 110 and 132.
// (codes that atma_linear_fp4_form returns)
enum Fp4Form { kFp4Ring16, kFp4Ring32, kFp4Kept16, kFp4Tile32, kFp4Tile64, kFp4Tile128, kFp4Tile256, kFp4Halves32, kFp4Halves64 };

static Fp4Form choose_fp4(const Fp4Args& a, bool gated) {
  Fp4Form best = kFp4Tile256;
  float least = 0.f;
  auto offer = [&](Fp4Form form, float us) {
    if (least == 0.f || us < least) best = form, least = us;
  };
  const float simds = 4.f * (float)device_cu_count();
  const int few_nk = (a.K + kFewBlock - 1) / kFewBlock;
  auto few = [&](Fp4Form form, const FewPlan& p, float fixed, float step, float block) {
    offer(form, fixed + step * (float)p.steps + block * (float)p.tiles * (float)p.groups * (float)few_nk / simds);
  };
  auto tile = [&](Fp4Form form, float fixed, const TileCost& c) {
    offer(form, fixed + tile_time(a.M, a.N, form >= kFp4Halves32 ? (a.nk + 1) / 2 : a.nk, c));
  };
  const bool some = a.M <= 1024;  // (beyond, tiles are ahead by far)
  if (gated) {
    if (some) few(kFp4Ring16, plan_few4<1, 2, 4, true, true>(a), 4.25f, 0.673f, 0.245f);
    tile(kFp4Halves64, 3.08f, {64, 64, 1.59f, 0.456f, 0.693f});
    tile(kFp4Tile128, 4.75f, {64, 128, 0.01f, 0.38f, 0.495f});
    tile(kFp4Tile256, 5.59f, {128, 256, 1.25f, 0.902f, 1.47f});
  } else {
    if (some) few(kFp4Ring16, plan_few4<1, 1, 4, true, false>(a), 3.68f, 0.483f, 0.198f);
    if (some) few(kFp4Ring32, plan_few4<2, 1, 4, true, false>(a), 4.34f, 0.818f, 0.189f);
    if (some && std::min<int64_t>(a.M, 16) * few_nk * 2 * kFewBlock <= kFewTokens)
      few(kFp4Kept16, plan_few4<1, 1, 8, false, false>(a), 4.57f, 0.297f, 0.225f);
    tile(kFp4Tile32, 4.15f, {128, 32, 0.f, 0.281f, 0.245f});
    tile(kFp4Tile64, 3.76f, {128, 64, 0.11f, 0.32f, 0.341f});
    tile(kFp4Halves32, 2.39f, {128, 32, 1.5f, 0.37f, 0.484f});
    tile(kFp4Halves64, 2.32f, {128, 64, 1.93f, 0.43f, 0.618f});
    tile(kFp4Tile128, 4.62f, {128, 128, 0.37f, 0.386f, 0.477f});
    tile(kFp4Tile256, 5.5f, {256, 256, 0.88f, 0.994f, 1.5f});
  }
  return best;
}

static bool fp4_sizes(int64_t M, int64_t rows, int64_t K) {
  return M >= 1 && M <= (1 << 30) && rows >= 1 && rows <= (1 << 28) && K >= kFp4Group && K <= (1 << 22) && K % kFp4Group == 0;
}

static int form_fp4(int64_t M, int64_t N, int64_t K, bool gated) {
  if (N > (1 << 28) || !fp4_sizes(M, gated ? 2 * N : N, K)) return -1;
  Fp4Args a{};
  a.M = M, a.N = N, a.K = (int)K, a.nk = (a.K + kFp4Block - 1) / kFp4Block;
  return choose_fp4(a, gated);
}

static int linear_fp4(const char* what, bool gated, Fp4Args a, int64_t K, int dtype, void* stream) {
  const int64_t rows = gated && a.N <= (1 << 28) ? 2 * a.N : a.N;
  if (dtype != ATMA_BF16 && dtype != ATMA_F16)
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: 16-bit activations (dtype %d)", what, dtype);
  if (a.M < 0 || !fp4_sizes(std::max<int64_t>(a.M, 1), rows, K))
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
  if (a.ldy < a.N) return set_error(ATMA_ERR_INVALID, "%s: rows of y must be at least N long", what);
  a.nk = (a.K + kFp4Block - 1) / kFp4Block;
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    const Fp4Form form = choose_fp4(a, gated);
    if (gated) {
      switch (form) {
        case kFp4Ring16: launch_few4<T, 1, 2, 4, true, true>(a, st); break;
        case kFp4Halves64: launch_tiles4<T, 2, 1, 2, 2, 3, true, 2>(a, st); break;
        case kFp4Tile128: launch_tiles4<T, 2, 2, 2, 2, 3, true>(a, st); break;
        default: launch_tiles4<T, 2, 4, 4, 2, 3, true>(a, st); break;
      }
    } else {
      switch (form) {
        case kFp4Ring16: launch_few4<T, 1, 1, 4, true, false>(a, st); break;
        case kFp4Ring32: launch_few4<T, 2, 1, 4, true, false>(a, st); break;
        case kFp4Kept16: launch_few4<T, 1, 1, 8, false, false>(a, st); break;
        case kFp4Tile32: launch_tiles4<T, 1, 1, 4, 1, 4, false>(a, st); break;
        case kFp4Tile64: launch_tiles4<T, 1, 2, 4, 1, 4, false>(a, st); break;
        case kFp4Halves32: launch_tiles4<T, 1, 1, 4, 1, 3, false, 2>(a, st); break;
        case kFp4Halves64: launch_tiles4<T, 1, 2, 4, 1, 3, false, 2>(a, st); break;
        case kFp4Tile128: launch_tiles4<T, 2, 2, 2, 2, 3, false>(a, st); break;
        default: launch_tiles4<T, 2, 4, 4, 2, 3, false>(a, st); break;
      }
    }
  };
  if (dtype == ATMA_BF16) launch(bf16{});
  else launch(f16{});
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

extern "C" int atma_linear_fp4_form(int64_t M, int64_t N, int64_t K) { return atma::form_fp4(M, N, K, false); }

extern "C" int atma_linear_gated_fp4_form(int64_t M, int64_t H, int64_t K) { return atma::form_fp4(M, H, K, true); }
