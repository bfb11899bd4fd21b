// Block-scaled 8-bit products: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]) for x (M, K) with a scale for each 128 values of
// a row and w (N, K) with a scale for each 128 x 128 block (fp8.h), and the MLP's first projection with its activation
// formed from the fp32 sums, h = gate * relu(a)^2, and quantized in the epilogue.  No reference counterpart.
//
// Products: v_mfma_scale_f32_16x16x128_f8f6f4, one instruction for each block of 128 along K.  Its scale operands carry
// the blocks' power-of-two scales (lane l: row l % 16), so the accumulator holds scaled sums from the first product on and
// no partial sum is ever rescaled.  Accumulators are fp32; inside the instruction the products of eight neighbouring k
// are aligned to the largest of them and keep about 14 bits below it (measured: 2^2 beside 2^16 is lost), which is 1.4e-5
// of the result for normally distributed values: far below the rounding to a 16-bit output, and the reason why there is
// no fp32 output.  The order of k inside a block is free (one scale covers it), so a lane takes whichever 16-byte pieces
// load best, the same ones of x and w.
#include <algorithm>
#include <type_traits>

#include "fp8.h"

namespace atma {

typedef int i32x8 __attribute__((ext_vector_type(8)));

union Frag8 {  // one operand: 32 values of a row
  i32x8 v;
  u32x4 q[2];
};

__device__ __forceinline__ f32x4 mfma_fp8(const Frag8& w, const Frag8& x, const f32x4& c, int ws, int xs) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, c, 0, 0, 0, ws, 0, xs);
}

struct Fp8Args {
  const uint8_t* x;  // (M, K), row stride ldx
  int64_t ldx;
  const uint8_t* xs;  // (M, nk), row stride ldxs, a multiple of 4
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

__device__ __forceinline__ float bias_at(const Fp8Args& a, int64_t n) {
  if (!a.bias) return 0.f;
  if (a.bias_dtype == ATMA_BF16) return to_f32(((const bf16*)a.bias)[n]);
  if (a.bias_dtype == ATMA_F16) return to_f32(((const f16*)a.bias)[n]);
  return ((const float*)a.bias)[n];
}

// relu(a)^2 * gate in fp32 (NaN passes through, as torch's relu)
__device__ __forceinline__ float gate_act(float av, float gv) {
  const float pos = av < 0.f ? 0.f : av;
  return gv * (pos * pos);
}

// ------------------------------------------------------------------------------------------------ tiles
// A workgroup of four waves, WF x WM, owns BF weight rows x BM tokens, a wave TF x TM tiles of 32 x 32
// (v_mfma_scale_f32_32x32x64_f8f6f4: two instructions for a block of 128 along K).  K runs in steps of 64 through a ring of
// NS stages in LDS, filled NS - 1 steps ahead by direct copies; the workgroup is persistent and the ring runs on across its
// tiles, so a tile's first copies fly during the last steps and the epilogue of the one before.  Everything else a tile
// reads -- the scales of four blocks at a time, the bias -- comes through the same copies into small rings of their own:
// the loop has no load into registers, whose wait would drain the ring.
//
// A step's rows are 64 bytes, four chunks of 16, chunk c of row r at position c ^ f(r): the 16 lanes that read one chunk of
// 16 rows cover all banks when f takes four values over the rows of each residue mod 4.  The weights are the MFMA's rows,
// in an order such that a lane's accumulators are 16 consecutive features of one token (row 8 q + 4 h + e is feature
// 16 h + 4 q + e; lane half h holds the rows 4 h + e of each 8): outputs are stored straight from registers.
__device__ __forceinline__ int x_swizzle(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int w_swizzle(int r) { return ((r >> 2) & 1) | (((r >> 4) & 1) << 1); }

template <int TF, int TM, int WF, int WM, int NS, bool GATED>
struct Fp8Tile {
  static constexpr int NW = WF * WM;
  static constexpr int BF = 32 * TF * WF, BM = 32 * TM * WM;
  static constexpr int OF = GATED ? BF / 2 : BF;  // output features
  static constexpr int TO = GATED ? TF / 2 : TF;  // tiles of output features a wave
  static constexpr int STAGE = (BF + BM) * 64;
  static constexpr int WCOPY = BF / 16 / NW, XCOPY = BM / 16 / NW;  // copies a wave and step: 16 rows each
  static constexpr int XS = BM > 64 ? BM : 64;                      // words of token scales
  static constexpr int AUX = (NS - 1) / 2 + 2;  // scale groups and tiles that can be under way (two steps at least each)
  static constexpr int LDS_AUX = NS * STAGE, LDS_BIAS = LDS_AUX + AUX * (XS + 64) * 4;
  static constexpr int LDS_TOP = LDS_BIAS + AUX * 1024, LDS = LDS_TOP + (GATED ? WF * BM * 4 : 0);
  static_assert(NW == 4 && BF % (16 * NW) == 0 && BF <= 256 && BM <= 256, "whole copies, a bias of 1 KiB");
  static_assert(BM % (16 * NW) == 0 || BM == 32, "whole copies");
  static_assert(!GATED || (OF == kFp8Block && TF == 2), "a gated tile is one block of output features");
  static_assert((NS - 2) * (WCOPY + XCOPY + 1) < 64, "vmcnt counts to 63");
};

template <typename C>
__device__ __forceinline__ bool fp8_tile_at(const Fp8Args& a, int xcd, int u, int64_t& m0, int64_t& f0) {
  const int t = xcd * a.per_xcd + u;
  if (u >= a.per_xcd || t >= a.m_tiles * a.f_tiles) return false;
  const int grp = t / (4 * a.f_tiles), r = t - grp * 4 * a.f_tiles;
  const int gm = min(4, a.m_tiles - 4 * grp);
  m0 = (int64_t)(4 * grp + r % gm) * C::BM;
  f0 = (int64_t)(r / gm) * C::OF;
  return true;
}

template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED>
__global__ void __launch_bounds__(64 * WF * WM, 2) fp8_tile_kernel(Fp8Args a) {
  using C = Fp8Tile<TF, TM, WF, WM, NS, GATED>;
  constexpr int TO = C::TO;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wm = wave / WF;
  const int r = lane & 31, h = lane >> 5;
  const int xcd = blockIdx.x & 7, nper = gridDim.x >> 3;
  const int steps = 2 * a.nk;
  int64_t m0, f0;
  int u = blockIdx.x >> 3;
  if (!fp8_tile_at<C>(a, xcd, u, m0, f0)) return;

  // ---- the copies, NS - 1 steps ahead of the products.  Copy i of a wave moves rows 16 (i NW + wave) .. + 15: lane l
  // writes row l / 4, position l % 4, and reads the chunk that belongs there; chunks past K (offset 2^31, past every tile)
  // and rows past the end read as zeros
  const uint32_t lds0 = lds_offset(lds);
  const int crow = lane >> 2;
  const int wk = 16 * ((lane & 3) ^ w_swizzle(16 * wave + crow)), xk = 16 * ((lane & 3) ^ x_swizzle(crow));
  const uint32_t wv0 = (uint32_t)(16 * wave + crow) * (uint32_t)a.ldw, xv0 = (uint32_t)(16 * wave + crow) * (uint32_t)a.ldx;
  const uint32_t wstep = 16u * C::NW * (uint32_t)a.ldw, xstep = 16u * C::NW * (uint32_t)a.ldx;
  __amdgpu_buffer_rsrc_t xr, wr, gr, xsr, wsr;
  int pu = u, pk = 0, pstage = 0, paux = 0, ptile = 0;
  int64_t pf0 = 0;
  bool pmore = true;
  auto aim = [&](int64_t tm0, int64_t tf0) {
    const int64_t rows = min((int64_t)C::BM, a.M - tm0);
    xr = buffer_rsrc(a.x + tm0 * a.ldx, (uint32_t)(rows * a.ldx));
    xsr = buffer_rsrc(a.xs + tm0 * a.ldxs, (uint32_t)(rows * a.ldxs));
    const uint32_t wb = (uint32_t)(min((int64_t)C::OF, a.N - tf0) * a.ldw);
    wr = buffer_rsrc(a.w + tf0 * a.ldw, wb);
    if constexpr (GATED) gr = buffer_rsrc(a.w + (a.N + tf0) * a.ldw, wb);
    const int64_t b0 = tf0 / kFp8Block;
    wsr = buffer_rsrc(a.ws + b0 * a.ldws, (uint32_t)((a.w_blocks - b0) * a.ldws));
    pf0 = tf0;
  };
  auto issue = [&]() {
    if (pk == 0 && a.bias && wave == C::NW - 2) {
      // 256 biases (gated: 128 of a, 128 of gate), in words, to this tile's slot
      const int size = a.bias_dtype == ATMA_F32 ? 4 : 2;
      const int64_t total = (GATED ? 2 : 1) * a.N * size;
      const __amdgpu_buffer_rsrc_t br = buffer_rsrc(a.bias, (uint32_t)((total + 3) & ~3ll));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int word = 64 * i + lane, f = word * 4 / size;  // the word's first feature in the tile
        if (64 * i * 4 / size < 256) {
          const int64_t n = pf0 + (GATED && f >= C::OF ? a.N + f - C::OF : f);
          dma_buf4(br, n * size < total ? (uint32_t)(n * size) : 0xfffffffcu, 0u,
                   lds + C::LDS_BIAS + 1024 * ptile + 256 * i);
        }
      }
    }
    if ((pk & 7) == 0) {
      const uint32_t slot = lds0 + C::LDS_AUX + paux * (C::XS + 64) * 4;
      const uint32_t k4 = (uint32_t)pk >> 1;
      if (wave < C::XS / 64)
        dma_buf4_at(xsr, (uint32_t)(64 * wave + lane) * (uint32_t)a.ldxs + k4, 0u, slot + 256 * wave);
      if (wave == C::NW - 1) {
        const uint32_t row = GATED ? (lane ? (uint32_t)(a.N / kFp8Block) : 0u) : (uint32_t)lane;
        dma_buf4_at(wsr, lane < 2 ? row * (uint32_t)a.ldws + k4 : 0x80000000u, 0u, slot + 4 * C::XS);
      }
      paux = paux + 1 == C::AUX ? 0 : paux + 1;
    }
    const uint32_t d = lds0 + pstage * C::STAGE + 1024 * wave;
    const int k = 64 * pk;
    const uint32_t wv = k + wk < a.K ? wv0 + (uint32_t)(k + wk) : 0x80000000u;
    const uint32_t xv = k + xk < a.K ? xv0 + (uint32_t)(k + xk) : 0x80000000u;
#pragma unroll
    for (int i = 0; i < C::WCOPY; ++i) {
      constexpr int half = C::WCOPY / 2;  // gated: the first half of a wave's copies are a rows, the others gate rows
      if (GATED && i >= half) dma_buf16_at(gr, wv + (i - half) * wstep, 0u, d + 1024 * C::NW * i);
      else dma_buf16_at(wr, wv + i * wstep, 0u, d + 1024 * C::NW * i);
    }
    if constexpr (C::XCOPY == 0) {
      if (wave < C::BM / 16) dma_buf16_at(xr, xv, 0u, d + C::BF * 64);
    }
#pragma unroll
    for (int i = 0; i < C::XCOPY; ++i) dma_buf16_at(xr, xv + i * xstep, 0u, d + C::BF * 64 + 1024 * C::NW * i);
    pstage = pstage + 1 == NS ? 0 : pstage + 1;
    if (++pk == steps) {
      int64_t nm0, nf0;
      pk = 0;
      ptile = ptile + 1 == C::AUX ? 0 : ptile + 1;
      pu += nper;
      pmore = fp8_tile_at<C>(a, xcd, pu, nm0, nf0);
      if (pmore) aim(nm0, nf0);
    }
  };

  // ---- operand reads
  const int wrow0 = 32 * TO * wf;  // the wave's first output feature in the tile
  const int wrow = 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
  uint32_t wofs[2], xofs[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    wofs[q] = (uint32_t)((wrow0 + wrow) * 64 + 16 * ((2 * h + q) ^ w_swizzle(wrow)));
    xofs[q] = (uint32_t)(C::BF * 64 + (32 * TM * wm + r) * 64 + 16 * ((2 * h + q) ^ x_swizzle(r)));
  }

  f32x16 acc[TF][TM];
  int stage = 0, aux = 0, tile = 0;
  aim(m0, f0);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (pmore) issue();
  while (true) {
    const uint32_t* words = nullptr;
    uint32_t xs[TM], ws[2];
    for (int k = 0; k < steps; k += 2) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        // this step's copies have landed in every wave, and every wave is done with the stage before it
        if (pmore) wait_vmcnt<(NS - 2) * (C::WCOPY + C::XCOPY)>();
        else wait_vmcnt<0>();
        lds_barrier();
        if (pmore) issue();
        if (s == 0) {
          if (k == 0) {
#pragma unroll
            for (int t = 0; t < TF; ++t) {
              float b[16] = {};
              const int f = wrow0 + 16 * h + (GATED ? t / TO * C::OF + 32 * (t % TO) : 32 * t);
              if (a.bias) {
                const uint8_t* slot = lds + C::LDS_BIAS + 1024 * tile;
                if (a.bias_dtype == ATMA_F32) {
#pragma unroll
                  for (int e = 0; e < 16; e += 4) {
                    const f32x4 v = *(const f32x4*)(slot + 4 * (f + e));
                    b[e] = v[0], b[e + 1] = v[1], b[e + 2] = v[2], b[e + 3] = v[3];
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < 16; e += 8) {
                    const u32x4 v = *(const u32x4*)(slot + 2 * (f + e));
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                      b[e + i] = a.bias_dtype == ATMA_BF16 ? elem16<bf16>(v, i) : elem16<f16>(v, i);
                  }
                }
              }
#pragma unroll
              for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][j][e] = b[e];
            }
            tile = tile + 1 == C::AUX ? 0 : tile + 1;
          }
          if ((k & 7) == 0) {
            words = (const uint32_t*)(lds + C::LDS_AUX + aux * (C::XS + 64) * 4);
            aux = aux + 1 == C::AUX ? 0 : aux + 1;
          }
          const int sh = 4 * (k & 7);  // byte (k / 2) % 4
#pragma unroll
          for (int j = 0; j < TM; ++j) xs[j] = words[32 * (TM * wm + j) + r] >> sh;
          ws[0] = words[C::XS + (GATED ? 0 : wrow0 / kFp8Block)] >> sh;
          ws[1] = GATED ? words[C::XS + 1] >> sh : 0;
        }
        const uint8_t* base = lds + stage * C::STAGE;
        stage = stage + 1 == NS ? 0 : stage + 1;
        Frag8 wv[TF], xv[TM];
#pragma unroll
        for (int t = 0; t < TF; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            wv[t].q[q] = *(const u32x4*)(base + wofs[q] + (GATED ? t / TO * (C::BF / 2) + 32 * (t % TO) : 32 * t) * 64);
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) xv[j].q[q] = *(const u32x4*)(base + xofs[q] + 32 * 64 * j);
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int t = 0; t < TF; ++t)
            acc[t][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                wv[t].v, xv[j].v, acc[t][j], 0, 0, 0, (int)ws[GATED ? t / TO : 0], 0, (int)xs[j]);
      }
    }

    // ---- epilogue of tile (m0, f0): token 32 (TM wm + j) + r, 16 consecutive features a tile
    if constexpr (!GATED) {
      const bool whole = f0 + C::OF <= a.N && a.ldy % 8 == 0;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int64_t m = m0 + 32 * (TM * wm + j) + r;
        if (m < a.M) {
#pragma unroll
          for (int t = 0; t < TF; ++t) {
            const int64_t n0 = f0 + wrow0 + 32 * t + 16 * h;
            T* y = (T*)a.y + m * a.ldy + n0;
            const f32x16& v = acc[t][j];
            if (whole) {
#pragma unroll
              for (int e = 0; e < 16; e += 8)
                *(u32x4*)(y + e) = u32x4{pack2<T>(v[e], v[e + 1]), pack2<T>(v[e + 2], v[e + 3]),
                                         pack2<T>(v[e + 4], v[e + 5]), pack2<T>(v[e + 6], v[e + 7])};
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (n0 + e < a.N) y[e] = from_f32<T>(v[e]);
            }
          }
        }
      }
    } else {
      // the activations in place of a's accumulators, their largest magnitude over the wave's features, then the tile's
      float* part = (float*)(lds + C::LDS_TOP);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = gate_act(acc[0][j][e], acc[1][j][e]);
          acc[0][j][e] = v;
          top = fmaxf(top, finite_abs(v));
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
        const float inv = fp8_inv_scale(code);
        const int64_t m = m0 + row;
        if (m < a.M) {
          if (wf == 0 && h == 0) a.ys[m * a.ldys + f0 / kFp8Block] = (uint8_t)code;
          const f32x16& v = acc[0][j];
          u32x4 o;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            o[q] = fp8_pack4(v[4 * q] * inv, v[4 * q + 1] * inv, v[4 * q + 2] * inv, v[4 * q + 3] * inv);
          *(u32x4*)((uint8_t*)a.y + m * a.ldy + f0 + wrow0 + 16 * h) = o;
        }
      }
    }
    u += nper;
    if (!fp8_tile_at<C>(a, xcd, u, m0, f0)) break;
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// At most 16 MT tokens: a stream of the weights.  A workgroup of NW waves owns FT tiles of 16 weight rows and its waves
// take the blocks of K in turn; operands come straight from memory in the MFMA's layout (32 bytes of a row a lane) and the
// waves' sums are joined through LDS in a fixed order.
template <typename T, int MT, int FT, int NW>
__global__ void __launch_bounds__(64 * NW) fp8_few_kernel(Fp8Args a) {
  __shared__ f32x4 red[NW][FT][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 16 * FT;
  const uint8_t* wp[FT];
  const uint8_t* xp[MT];
  const uint8_t* xsp[MT];
#pragma unroll
  for (int t = 0; t < FT; ++t) wp[t] = a.w + min(f0 + 16 * t + r, a.N - 1) * a.ldw;
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = min((int64_t)(16 * j + r), a.M - 1);
    xp[j] = a.x + m * a.ldx;
    xsp[j] = a.xs + m * a.ldxs;
  }
  const uint8_t* wsp = a.ws + f0 / kFp8Block * a.ldws;
  f32x4 acc[FT][MT] = {};
  for (int kb = wave; kb < a.nk; kb += NW) {
    Frag8 wv[FT], xv[MT];
    int xsc[MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = kb * kFp8Block + 32 * g + 16 * h;
      const bool in = k < a.K;
#pragma unroll
      for (int t = 0; t < FT; ++t) wv[t].q[h] = in ? *(const u32x4*)(wp[t] + k) : u32x4{};
#pragma unroll
      for (int j = 0; j < MT; ++j) xv[j].q[h] = in ? *(const u32x4*)(xp[j] + k) : u32x4{};
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) xsc[j] = xsp[j][kb];
    const int wsc = wsp[kb];
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[t][j] = mfma_fp8(wv[t], xv[j], acc[t][j], wsc, xsc[j]);
  }
#pragma unroll
  for (int t = 0; t < FT; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[wave][t][j][lane] = acc[t][j];
  __syncthreads();
  for (int i = wave; i < FT * MT; i += NW) {
    const int t = i / MT, j = i % MT;
    f32x4 s = red[0][t][j][lane];
    for (int q = 1; q < NW; ++q) s += red[q][t][j][lane];
    const int64_t n0 = f0 + 16 * t + 4 * g, m = 16 * j + r;
    if (m >= a.M) continue;
    T* y = (T*)a.y + m * a.ldy + n0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n0 + e < a.N) y[e] = from_f32<T>(s[e] + bias_at(a, n0 + e));
  }
}

// The gated form: a workgroup of 16 waves owns one block of 128 output features; wave w takes their tile w % 8 (its a and
// gate rows) and the blocks of K of parity w / 8.
template <int MT>
__global__ void __launch_bounds__(1024) fp8_few_gated_kernel(Fp8Args a) {
  __shared__ f32x4 red[8][2][MT][64];
  __shared__ float top[8][16 * MT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = wave & 7, part = wave >> 3;
  const int r = lane & 15, g = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * kFp8Block;
  const uint8_t* wp[2];
  const uint8_t* wsp[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    wp[t] = a.w + (t * a.N + f0 + 16 * tile + r) * a.ldw;
    wsp[t] = a.ws + (t * a.N + f0) / kFp8Block * a.ldws;
  }
  const uint8_t* xp[MT];
  const uint8_t* xsp[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = min((int64_t)(16 * j + r), a.M - 1);
    xp[j] = a.x + m * a.ldx;
    xsp[j] = a.xs + m * a.ldxs;
  }
  f32x4 acc[2][MT] = {};
  for (int kb = part; kb < a.nk; kb += 2) {
    Frag8 wv[2], xv[MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = kb * kFp8Block + 32 * g + 16 * h;
      const bool in = k < a.K;
#pragma unroll
      for (int t = 0; t < 2; ++t) wv[t].q[h] = in ? *(const u32x4*)(wp[t] + k) : u32x4{};
#pragma unroll
      for (int j = 0; j < MT; ++j) xv[j].q[h] = in ? *(const u32x4*)(xp[j] + k) : u32x4{};
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[t][j] = mfma_fp8(wv[t], xv[j], acc[t][j], wsp[t][kb], xsp[j][kb]);
  }
  if (part == 1) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < MT; ++j) red[tile][t][j][lane] = acc[t][j];
  }
  __syncthreads();
  const int64_t n0 = f0 + 16 * tile + 4 * g;
  if (part == 0) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const f32x4 sa = acc[0][j] + red[tile][0][j][lane], sg = acc[1][j] + red[tile][1][j][lane];
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float h = gate_act(sa[e] + bias_at(a, n0 + e), sg[e] + bias_at(a, a.N + n0 + e));
        acc[0][j][e] = h;
        m = fmaxf(m, finite_abs(h));
      }
      m = fmaxf(m, wave_xor(m, 16));
      m = fmaxf(m, wave_xor(m, 32));
      if (g == 0) top[tile][16 * j + r] = m;
    }
  }
  __syncthreads();
  if (part == 0) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int64_t m = 16 * j + r;
      if (m >= a.M) continue;
      float t = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) t = fmaxf(t, top[q][16 * j + r]);
      const int code = fp8_scale_code(t);
      const float inv = fp8_inv_scale(code);
      const f32x4& h = acc[0][j];
      *(uint32_t*)((uint8_t*)a.y + m * a.ldy + n0) = fp8_pack4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
      if (tile == 0 && g == 0) a.ys[m * a.ldys + f0 / kFp8Block] = (uint8_t)code;
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
template <typename T, int TF, int TM, int WF, int WM, int NS, bool GATED>
static void launch_tiles(Fp8Args a, hipStream_t s) {
  using C = Fp8Tile<TF, TM, WF, WM, NS, GATED>;
  a.m_tiles = (int)((a.M + C::BM - 1) / C::BM);
  a.f_tiles = (int)((a.N + C::OF - 1) / C::OF);
  const int64_t tiles = (int64_t)a.m_tiles * a.f_tiles;
  a.per_xcd = (int)((tiles + 7) / 8);
  constexpr int per_cu = std::min(4, 160 * 1024 / C::LDS);  // workgroups that fit a CU's LDS
  const int64_t wgs = std::min<int64_t>((int64_t)device_cu_count() / 8 * 8 * per_cu, 8 * (int64_t)a.per_xcd);
  fp8_tile_kernel<T, TF, TM, WF, WM, NS, GATED><<<dim3((unsigned)wgs), dim3(64 * C::NW), 0, s>>>(a);
}

// Checks shared by the products; rows: weight rows (N, or 2 N gated)
static int check_fp8(const char* what, const Fp8Args& a, int64_t rows) {
  if (a.M < 0 || a.N < 1 || a.K < 16 || a.K % 16 || a.K > (1 << 22) || a.M > (1 << 30) || rows > (1 << 28))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: unsupported shape M=%lld N=%lld K=%d (K a multiple of 16)", what,
                     (long long)a.M, (long long)a.N, a.K);
  if (a.M == 0) return ATMA_OK;
  if (!a.x || !a.xs || !a.w || !a.ws || !a.y) return set_error(ATMA_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)a.x % 16 || a.ldx % 16 || a.ldx < a.K || (uintptr_t)a.w % 16 || a.ldw % 16 || a.ldw < a.K)
    return set_error(ATMA_ERR_INVALID, "%s: rows of x and w must be 16-byte aligned and at least K long", what);
  if ((uintptr_t)a.xs % 4 || a.ldxs % 4 || a.ldxs < a.nk || (uintptr_t)a.ws % 4 || a.ldws % 4 || a.ldws < a.nk)
    return set_error(ATMA_ERR_INVALID, "%s: rows of scales must be 4-byte aligned and hold %d", what, a.nk);
  // a tile's rows (at most 256) are addressed by 32-bit byte offsets
  if (a.ldx > (1 << 23) || a.ldw > (1 << 23))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: rows more than 8 MiB apart", what);
  if (a.ldxs > (1 << 20) || a.w_blocks * a.ldws >= (1ll << 31))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: scales too far apart", what);
  if (a.bias && (uintptr_t)a.bias % 4) return set_error(ATMA_ERR_INVALID, "%s: bias must be 4-byte aligned", what);
  if (a.bias && !dtype_size(a.bias_dtype))
    return set_error(ATMA_ERR_UNSUPPORTED, "%s: bias in fp32 or 16 bits (dtype %d)", what, a.bias_dtype);
  return ATMA_OK;
}

template <typename T>
static void launch_linear(const Fp8Args& a, hipStream_t s) {
  if (a.M <= 16) {
    fp8_few_kernel<T, 1, 1, 8><<<dim3((unsigned)((a.N + 15) / 16)), 512, 0, s>>>(a);
  } else if (a.M <= 32) {
    fp8_few_kernel<T, 2, 1, 8><<<dim3((unsigned)((a.N + 15) / 16)), 512, 0, s>>>(a);
  } else if (((a.M + 127) / 128) * ((a.N + 255) / 256) >= 2 * device_cu_count()) {
    launch_tiles<T, 2, 4, 4, 1, 3, false>(a, s);
  } else if (((a.M + 127) / 128) * ((a.N + 127) / 128) >= device_cu_count()) {
    launch_tiles<T, 2, 2, 2, 2, 4, false>(a, s);
  } else {
    launch_tiles<T, 1, 1, 2, 2, 8, false>(a, s);
  }
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
  if (ldy < N || (uintptr_t)y % 2 || (ldy % 8 == 0 && (uintptr_t)y % 16))
    return set_error(ATMA_ERR_INVALID, "linear_fp8: rows of y must be at least N long, 16-byte aligned where ldy %% 8 == 0");
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
  hipStream_t s = (hipStream_t)stream;
  if (M <= 16) fp8_few_gated_kernel<1><<<dim3((unsigned)(H / kFp8Block)), 1024, 0, s>>>(a);
  else if (M <= 32) fp8_few_gated_kernel<2><<<dim3((unsigned)(H / kFp8Block)), 1024, 0, s>>>(a);
  else if (((M + 127) / 128) * (H / kFp8Block) >= 2 * device_cu_count()) launch_tiles<bf16, 2, 4, 4, 1, 3, true>(a, s);
  else if (((M + 63) / 64) * (H / kFp8Block) >= device_cu_count()) launch_tiles<bf16, 2, 2, 4, 1, 3, true>(a, s);
  else launch_tiles<bf16, 2, 1, 4, 1, 4, true>(a, s);
  return check_launch("linear_gated_fp8");
}
