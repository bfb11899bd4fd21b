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
// Chunk position of a tile's row in LDS: rows are 128 bytes, 8 chunks of 16, chunk c of row r at position c ^ f(r).  The
// 16 lanes that read one chunk of 16 rows cover all banks when f takes 8 values over the rows of each parity: 16
// consecutive token rows; weight rows 16 a + 4 t + b, a, b < 4 (the order below), or 8 a + 4 t + b.
__device__ __forceinline__ int x_swizzle(int r) { return (r >> 1) & 7; }
template <int G>
__device__ __forceinline__ int w_swizzle(int r) {
  if constexpr (G == 4) return ((r >> 1) & 1) | (((r >> 4) & 3) << 1);
  else if constexpr (G == 2) return ((r >> 1) & 1) | (((r >> 3) & 3) << 1);
  else return (r >> 1) & 7;
}

// A workgroup of WF x WM waves owns BF weight rows x BM tokens and a wave TF x TM tiles of 16 x 16.  The weights are the
// MFMA's rows: their order inside a wave's rows is chosen such that a lane's accumulators of G tiles are 4 G consecutive
// features of one token (tile t's row 4 a + b is feature 4 G a + 4 t + b), stored straight from registers.
template <typename T, int TF, int TM, int WF, int WM, bool GATED>
struct Fp8Tile {
  static constexpr int NW = WF * WM;
  static constexpr int BF = 16 * TF * WF, BM = 16 * TM * WM;
  static constexpr int OF = GATED ? BF / 2 : BF;   // output features
  static constexpr int TO = GATED ? TF / 2 : TF;   // tiles of output features a wave
  static constexpr int G = TO < 4 ? TO : 4;
  static constexpr int STAGE = (BF + BM) * kFp8Block;
  static constexpr int WCOPY = BF / 8 / NW, XCOPY = BM / 8 / NW;  // copies a wave and step: 8 rows each
  static_assert(BF % (8 * NW) == 0 && BM % (8 * NW) == 0 && (NW == 4 || NW == 8), "whole copies");
  static_assert(!GATED || OF == kFp8Block, "a gated tile is one block of output features");
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

template <typename T, int TF, int TM, int WF, int WM, bool GATED>
__global__ void __launch_bounds__(64 * WF * WM) fp8_tile_kernel(Fp8Args a) {
  using C = Fp8Tile<T, TF, TM, WF, WM, GATED>;
  constexpr int G = C::G, TO = C::TO;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * C::STAGE];
  __shared__ float amax_part[GATED ? WF : 1][GATED ? C::BM : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wm = wave / WF;
  const int r = lane & 15, g = lane >> 4;
  const int xcd = blockIdx.x & 7, nper = gridDim.x >> 3;
  int64_t m0, f0;
  int u = blockIdx.x >> 3;
  if (!fp8_tile_at<C>(a, xcd, u, m0, f0)) return;

  // ---- copies: instruction i of a wave moves rows 8 (i NW + wave) .. + 7 of a tile; lane l writes row l / 8, position
  // l % 8, and reads the chunk that belongs there; chunks past K (offset 2^31, past every tile) and rows past the end
  // read as zeros
  const int crow = lane >> 3, cpos = lane & 7;
  auto row_of = [&](int i) { return 8 * (i * C::NW + wave) + crow; };
  __amdgpu_buffer_rsrc_t xr, wr, gr;
  auto aim = [&](int64_t tm0, int64_t tf0) {
    xr = buffer_rsrc(a.x + tm0 * a.ldx, (uint32_t)(min((int64_t)C::BM, a.M - tm0) * a.ldx));
    const uint32_t wb = (uint32_t)(min((int64_t)C::OF, a.N - tf0) * a.ldw);
    wr = buffer_rsrc(a.w + tf0 * a.ldw, wb);
    if constexpr (GATED) gr = buffer_rsrc(a.w + (a.N + tf0) * a.ldw, wb);
  };
  const uint32_t lds0 = lds_offset(lds);
  auto issue = [&](int stage, int kb) {
    const uint32_t d = lds0 + stage * C::STAGE + 1024 * wave;
#pragma unroll
    for (int i = 0; i < C::WCOPY; ++i) {
      const int row = row_of(i);
      const int k = kb * kFp8Block + 16 * (cpos ^ w_swizzle<G>(row));
      const int half = GATED ? C::BF / 2 : C::BF;
      const bool second = GATED && 8 * i * C::NW >= half;
      const uint32_t v = k < a.K ? (uint32_t)(row - (second ? half : 0)) * (uint32_t)a.ldw + (uint32_t)k : 0x80000000u;
      dma_buf16_at(second ? gr : wr, v, 0u, d + 1024 * C::NW * i);
    }
#pragma unroll
    for (int i = 0; i < C::XCOPY; ++i) {
      const int row = row_of(i);
      const int k = kb * kFp8Block + 16 * (cpos ^ x_swizzle(row));
      const uint32_t v = k < a.K ? (uint32_t)row * (uint32_t)a.ldx + (uint32_t)k : 0x80000000u;
      dma_buf16_at(xr, v, 0u, d + C::BF * kFp8Block + 1024 * C::NW * i);
    }
  };

  // ---- scales of the wave's tokens and weight blocks, four steps a word
  uint32_t xs_next[TM], ws_next[2];
  const int wrow0 = 16 * TO * wf;  // the wave's first output feature in the tile
  auto load_scales = [&](int64_t tm0, int64_t tf0, int kb) {
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int64_t m = min(tm0 + 16 * (TM * wm + t) + r, a.M - 1);
      xs_next[t] = *(const uint32_t*)(a.xs + m * a.ldxs + kb);
    }
    const int64_t wb = min(tf0 + wrow0, a.N - 1) / kFp8Block;
    ws_next[0] = *(const uint32_t*)(a.ws + wb * a.ldws + kb);
    if constexpr (GATED) ws_next[1] = *(const uint32_t*)(a.ws + (a.N / kFp8Block + wb) * a.ldws + kb);
  };

  // ---- operand reads
  uint32_t wofs[TF][2], xofs[2];
#pragma unroll
  for (int t = 0; t < TF; ++t) {
    const int to = t % TO, grp = to / G;  // tile to of the a half or the gate half
    const int row = (t / TO) * (C::BF / 2) + wrow0 + 16 * G * grp + 4 * G * (r >> 2) + 4 * (to % G) + (r & 3);
#pragma unroll
    for (int h = 0; h < 2; ++h) wofs[t][h] = row * kFp8Block + 16 * ((g + 4 * h) ^ w_swizzle<G>(row));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    xofs[h] = C::BF * kFp8Block + (16 * TM * wm + r) * kFp8Block + 16 * ((g + 4 * h) ^ x_swizzle(r));

  f32x4 acc[TF][TM];
  uint32_t xs_now[TM], ws_now[2];
  int stage = 0;
  aim(m0, f0);
  load_scales(m0, f0, 0);
  issue(0, 0);
  while (true) {
#pragma unroll
    for (int t = 0; t < TF; ++t)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[t][j] = f32x4{};
    int64_t nm0 = 0, nf0 = 0;
    bool more = false;
    for (int kb = 0; kb < a.nk; ++kb) {
      // the copies of this step have landed in every wave, and every wave is done with the other stage
      wait_vmcnt<0>();
      if ((kb & 3) == 0) {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          xs_now[j] = xs_next[j];
          asm volatile("" : "+v"(xs_now[j]));  // the compiler's own wait belongs here, before the next copies
        }
        ws_now[0] = ws_next[0];
        ws_now[1] = GATED ? ws_next[1] : 0;
        asm volatile("" : "+v"(ws_now[0]), "+v"(ws_now[1]));
      }
      lds_barrier();
      if (kb + 1 < a.nk) {
        if (((kb + 1) & 3) == 0) load_scales(m0, f0, kb + 1);
        issue(stage ^ 1, kb + 1);
      } else {
        u += nper;
        more = fp8_tile_at<C>(a, xcd, u, nm0, nf0);
        if (more) {
          aim(nm0, nf0);
          load_scales(nm0, nf0, 0);
          issue(stage ^ 1, 0);
        }
      }
      const uint8_t* base = lds + stage * C::STAGE;
      const int sh = 8 * (kb & 3);
      Frag8 wv[TF];
#pragma unroll
      for (int t = 0; t < TF; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) wv[t].q[h] = *(const u32x4*)(base + wofs[t][h]);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        Frag8 xv;
#pragma unroll
        for (int h = 0; h < 2; ++h) xv.q[h] = *(const u32x4*)(base + xofs[h] + 16 * j * kFp8Block);
        const int xsc = (int)(xs_now[j] >> sh);
#pragma unroll
        for (int t = 0; t < TF; ++t)
          acc[t][j] = mfma_fp8(wv[t], xv, acc[t][j], (int)(ws_now[GATED ? t / TO : 0] >> sh), xsc);
      }
      stage ^= 1;
    }

    // ---- epilogue of tile (m0, f0): token 16 (TM wm + j) + r, features 4 G consecutive per group of tiles
    if constexpr (!GATED) {
      const bool whole = f0 + C::OF <= a.N && a.ldy % 8 == 0;
#pragma unroll
      for (int grp = 0; grp < TO / G; ++grp) {
        const int64_t n0 = f0 + wrow0 + 16 * G * grp + 4 * G * g;
        float b[4 * G];
#pragma unroll
        for (int e = 0; e < 4 * G; ++e) b[e] = n0 + e < a.N ? bias_at(a, n0 + e) : 0.f;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int64_t m = m0 + 16 * (TM * wm + j) + r;
          if (m >= a.M) continue;
          T* y = (T*)a.y + m * a.ldy + n0;
          float v[4 * G];
#pragma unroll
          for (int e = 0; e < 4 * G; ++e) v[e] = acc[grp * G + e / 4][j][e & 3] + b[e];
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4 * G; e += 8)
              *(u32x4*)(y + e) = u32x4{pack2<T>(v[e], v[e + 1]), pack2<T>(v[e + 2], v[e + 3]),
                                       pack2<T>(v[e + 4], v[e + 5]), pack2<T>(v[e + 6], v[e + 7])};
          } else {
#pragma unroll
            for (int e = 0; e < 4 * G; ++e)
              if (n0 + e < a.N) y[e] = from_f32<T>(v[e]);
          }
        }
      }
    } else {
      // the activations, in place of the a half's accumulators, and their largest magnitude over the wave's features
      float top[TM] = {};
#pragma unroll
      for (int t = 0; t < TO; ++t) {
        const int64_t n0 = f0 + wrow0 + 16 * G * (t / G) + 4 * G * g + 4 * (t % G);
        float ba[4], bg[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ba[e] = bias_at(a, n0 + e), bg[e] = bias_at(a, a.N + n0 + e);
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float h = gate_act(acc[t][j][e] + ba[e], acc[TO + t][j][e] + bg[e]);
            acc[t][j][e] = h;
            top[j] = fmaxf(top[j], finite_abs(h));
          }
      }
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        top[j] = fmaxf(top[j], wave_xor(top[j], 16));
        top[j] = fmaxf(top[j], wave_xor(top[j], 32));
        if (g == 0) amax_part[wf][16 * (TM * wm + j) + r] = top[j];
      }
      lds_barrier();
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int row = 16 * (TM * wm + j) + r;
        float t = amax_part[0][row];
#pragma unroll
        for (int q = 1; q < WF; ++q) t = fmaxf(t, amax_part[q][row]);
        const int code = fp8_scale_code(t);
        const float inv = fp8_inv_scale(code);
        const int64_t m = m0 + row;
        if (m >= a.M) continue;
        if (wf == 0 && g == 0) a.ys[m * a.ldys + f0 / kFp8Block] = (uint8_t)code;
#pragma unroll
        for (int grp = 0; grp < TO / G; ++grp) {
          uint32_t o[G];
#pragma unroll
          for (int t4 = 0; t4 < G; ++t4) {
            const f32x4& h = acc[grp * G + t4][j];
            o[t4] = fp8_pack4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
          }
          uint8_t* y = (uint8_t*)a.y + m * a.ldy + f0 + wrow0 + 16 * G * grp + 4 * G * g;
          if constexpr (G == 4) *(u32x4*)y = u32x4{o[0], o[1], o[2], o[3]};
          else if constexpr (G == 2) *(u32x2*)y = u32x2{o[0], o[1]};
          else *(uint32_t*)y = o[0];
        }
      }
    }
    if (!more) break;
    m0 = nm0;
    f0 = nf0;
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
template <typename T, int TF, int TM, int WF, int WM, bool GATED>
static void launch_tiles(Fp8Args a, hipStream_t s) {
  using C = Fp8Tile<T, TF, TM, WF, WM, GATED>;
  a.m_tiles = (int)((a.M + C::BM - 1) / C::BM);
  a.f_tiles = (int)((a.N + C::OF - 1) / C::OF);
  const int64_t tiles = (int64_t)a.m_tiles * a.f_tiles;
  a.per_xcd = (int)((tiles + 7) / 8);
  const int per_cu = 160 * 1024 / (2 * C::STAGE + 4096);  // workgroups that fit a CU's LDS
  const int64_t wgs = std::min<int64_t>((int64_t)device_cu_count() / 8 * 8 * std::max(per_cu, 1), 8 * (int64_t)a.per_xcd);
  fp8_tile_kernel<T, TF, TM, WF, WM, GATED><<<dim3((unsigned)wgs), dim3(64 * C::NW), 0, s>>>(a);
}

// Checks shared by the products; rows: weight rows (N, or 2 N gated)
static int check_fp8(const char* what, const Fp8Args& a, int64_t rows) {
  if (a.M < 0 || a.N < 1 || a.K < 16 || a.K % 16 || a.K > (1 << 22) || a.M > (1 << 30) || rows > (1 << 30))
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
  if (a.bias && (uintptr_t)a.bias % (size_t)std::max(dtype_size(a.bias_dtype), 1))
    return set_error(ATMA_ERR_INVALID, "%s: unaligned bias", what);
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
  } else if (((a.M + 255) / 256) * ((a.N + 255) / 256) >= device_cu_count()) {
    launch_tiles<T, 4, 8, 4, 2, false>(a, s);
  } else {
    launch_tiles<T, 4, 4, 2, 2, false>(a, s);
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
  Fp8Args a{(const uint8_t*)x, ldx, (const uint8_t*)xs, ldxs, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws, bias,
            bias_dtype, y, ldy, nullptr, 0, M, N, (int)K, (int)((K + kFp8Block - 1) / kFp8Block), 0, 0, 0};
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
  Fp8Args a{(const uint8_t*)x, ldx, (const uint8_t*)xs, ldxs, (const uint8_t*)w, ldw, (const uint8_t*)ws, ldws, bias,
            bias_dtype, y, ldy, (uint8_t*)ys, ldys, M, H, (int)K, (int)((K + kFp8Block - 1) / kFp8Block), 0, 0, 0};
  if (H < kFp8Block || H % kFp8Block || H > (1 << 29))
    return set_error(ATMA_ERR_UNSUPPORTED, "linear_gated_fp8: H must be a multiple of %d (got %lld)", kFp8Block,
                     (long long)H);
  if (const int rc = check_fp8("linear_gated_fp8", a, 2 * H)) return rc;
  if (M == 0) return ATMA_OK;
  if (!ys || (uintptr_t)y % 16 || ldy % 16 || ldy < H || ldys < H / kFp8Block)
    return set_error(ATMA_ERR_INVALID, "linear_gated_fp8: rows of y must be 16-byte aligned and at least H long");
  hipStream_t s = (hipStream_t)stream;
  if (M <= 16) fp8_few_gated_kernel<1><<<dim3((unsigned)(H / kFp8Block)), 1024, 0, s>>>(a);
  else if (M <= 32) fp8_few_gated_kernel<2><<<dim3((unsigned)(H / kFp8Block)), 1024, 0, s>>>(a);
  else if (((M + 255) / 256) * (H / kFp8Block) >= device_cu_count()) launch_tiles<bf16, 4, 8, 4, 2, true>(a, s);
  else launch_tiles<bf16, 4, 4, 4, 1, true>(a, s);
  return check_launch("linear_gated_fp8");
}
