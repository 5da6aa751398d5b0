// tile8.h -- a tile of a product of rows in 8 bits with weights in 8 bits, on the
// matrix instructions of gfx950 (internal; multiply8.hip says how it works, and
// what it measured).
#pragma once

#include "experts.h"

namespace ien {
namespace {

typedef int int8v __attribute__((ext_vector_type(8)));

struct Args8 {
  const uint8_t *x;
  long xs;
  const uint8_t *scales;
  long ss;
  int taps, cb, step;
  long images, H, W, OH, OW;  // rows: 1 map of 1 x rows
  long row0, rows;
  const uint8_t *w;
  const uint32_t *ws;
  const float *bias;
  long n, npad;
  void *y;
  long ys;
  int f32, exact, act;  // f32 outputs, sums in f32 (f32 outputs always)
  const void *add;
  long as;
  int image;  // a map's pixels
  int tiles_m, tiles_n, ksplit, kchunks;
  float *part;
  int *tile_count;
  // Experts: the tiles of a plan and how many, the pairs in the order of their
  // experts (of `top` a token), panels of weights an expert, rows in 8 bits out.
  const ExpertTile *list;
  const int *total, *order;
  int top;
  uint8_t *q, *qs;
  long qstride, qsstride;
};

// What a launch multiplies, and into what: rows or a map's pixels into rows; the
// plan's rows (ROWS) into rows; their tokens' rows into rows in 8 bits, an
// activation of each output (ACT) or of every first 32 of 64 that the others are
// multiplied by (GATED).
enum Kind8 { PLAIN8, EXPERTS_ROWS8, EXPERTS_ACT8, EXPERTS_GATED8 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight e4m3 bytes under a scale as bf16.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A tile of a launch: FM x FN blocks of 32 rows x 32 outputs a wave, WM x WN
// waves, a ring of S stages in LDS, each a block of 128 deep of the tile's
// rows and weights and their scales.
template <int FM_, int FN_, int WM_, int WN_, int S_>
struct Tile8 {
  static constexpr int FM = FM_, FN = FN_, WM = WM_, WN = WN_, S = S_;
  static constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int B0 = TM * BLOCK8, SX0 = B0 + TN * BLOCK8, SW0 = SX0 + TM * 4;
  static constexpr int A_LOADS = TM / 8 / WAVES, B_LOADS = TN / 8 / WAVES;  // a wave and stage, 1 KiB each
  static constexpr int S_PIECES = (TM + TN) / 64, S_LOADS = (S_PIECES + WAVES - 1) / WAVES;  // 256 bytes each
  static constexpr int STAGE = SX0 + WAVES * S_LOADS * 256;
  static constexpr int LOADS = A_LOADS + B_LOADS + S_LOADS;
  static constexpr int PITCH = 32 * FN + 4;  // floats between the epilogue's rows
  static constexpr int STAGING = WM * WN * 32 * PITCH * 4;
  static constexpr int BIAS0 = S * STAGE > STAGING ? S * STAGE : STAGING;
  static constexpr int LDS = BIAS0 + TN * 4;
  static_assert(A_LOADS * 8 * WAVES == TM && B_LOADS * 8 * WAVES == TN, "loads a wave");
};

// Buffer loads into LDS (dma_lds) with the place as a wave's base and a
// constant, and a uniform offset beside the lane's: 16 bytes a lane, or a byte
// a lane, each in a dword of LDS.
template <int CONST>
__device__ __forceinline__ void dma16_at(int4v rsrc, unsigned wave_base, int off, int soff) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds"
               :: "s"(wave_base), "n"(CONST), "v"(off), "s"(rsrc), "s"(soff) : "memory", "m0", "scc");
}
template <int CONST>
__device__ __forceinline__ void dma1_at(int4v rsrc, unsigned wave_base, int off, int soff) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_ubyte %2, %3, %4 offen lds"
               :: "s"(wave_base), "n"(CONST), "v"(off), "s"(rsrc), "s"(soff) : "memory", "m0", "scc");
}

// How many of n things are done before step k of `steps`.
constexpr int share8(int k, int n, int steps) { return k >= steps ? n : k * n / steps; }

// f(Const<0>) .. f(Const<N - 1>).
template <int V>
struct Const {
  static constexpr int value = V;
  constexpr operator int() const { return V; }
};
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (I < N) {
    f(Const<I>{});
    each<N, I + 1>(f);
  }
}

// A tile's outputs as rows in 8 bits.  The products are weights x rows, so a lane
// holds 16 of every 32 outputs of one row: biases, activation, gate and the largest
// magnitude are its own, the other 16 outputs the lane's 32 further on, and where a
// wave has half a block's outputs the other half is the wave's beside it (a word of
// LDS a row).  The bytes go through LDS for 16 of them a lane.
template <typename T, bool GATED>
__device__ __forceinline__ void into_rows8(const Args8 &a, floatx16 (&acc)[T::FM][T::FN], unsigned char *lds, long m0,
                                           long rows, long n0, int tid) {
  constexpr int COLS = 32 * T::FN, OUTS = GATED ? COLS / 2 : COLS, JS = OUTS / 32;  // a wave's columns and outputs
  constexpr bool SHARED = OUTS == 64;  // a block of 128 is two waves'
  static_assert((OUTS == 128 || (SHARED && T::WN == 2)) && T::FN % 2 == 0, "blocks of outputs");
  constexpr int PITCH = OUTS + 16, PIECES = OUTS / 16;
  constexpr int MAX0 = T::WAVES * 32 * PITCH;  // floats [wn][row]
  static_assert(MAX0 + T::WN * T::TM * 4 <= T::BIAS0, "the epilogue's LDS");
  const int lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % T::WM, wn = wave / T::WM;
  const float *bias = (const float *)(lds + T::BIAS0) + wn * COLS + 4 * hi;
  float *maxima = (float *)(lds + MAX0);
  const long out0 = (GATED ? n0 / 2 : n0) + wn * OUTS;  // this wave's first output
  float largest[T::FM];
  const bool ragged = out0 + OUTS > a.n;
  with_act8(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < T::FM; i++) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < JS; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const float4v b = *(const float4v *)(bias + 32 * (GATED ? 2 * j : j) + 8 * q);
          float4v u{};
          if constexpr (GATED) u = *(const float4v *)(bias + 32 * (2 * j + 1) + 8 * q);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int r = 4 * q + e;
            float v = act8<decltype(act)::value>(acc[i][GATED ? 2 * j : j][r] + b[e]);
            if constexpr (GATED) v *= acc[i][2 * j + 1][r] + u[e];
            acc[i][j][r] = v;
            m = fmaxf(m, fabsf(v));  // (a NaN is passed over)
          }
        }
      largest[i] = m;
    }
  });
  // What is rare: outputs past the last one, which are zeros, and infinities, which are NaN and no largest magnitude.
  bool infinite = false;
#pragma unroll
  for (int i = 0; i < T::FM; i++) infinite = infinite || !finite8(largest[i]);
  if (ragged || __ballot(infinite)) {
#pragma unroll
    for (int i = 0; i < T::FM; i++) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < JS; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          float v = acc[i][j][r];
          if (out0 + 32 * j + 8 * (r / 4) + 4 * hi + r % 4 >= a.n) v = 0.0f;
          if (!finite8(v)) v = __uint_as_float(0x7fc00000);
          acc[i][j][r] = v;
          m = fmaxf(m, fabsf(v));
        }
      largest[i] = m;
    }
  }
#pragma unroll
  for (int i = 0; i < T::FM; i++) largest[i] = fmaxf(largest[i], __shfl_xor(largest[i], 32));
  if constexpr (SHARED) {
#pragma unroll
    for (int i = 0; i < T::FM; i++)
      if (hi == 0) maxima[wn * T::TM + (wm * T::FM + i) * 32 + l32] = largest[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::FM; i++)
      largest[i] = fmaxf(largest[i], maxima[(wn ^ 1) * T::TM + (wm * T::FM + i) * 32 + l32]);
  }
  const int block = (int)(out0 / BLOCK8);
  if ((long)block * BLOCK8 >= a.n) return;
  unsigned char *st = lds + wave * 32 * PITCH;
#pragma unroll
  for (int i = 0; i < T::FM; i++) {
    const long r0 = m0 + (wm * T::FM + i) * 32;
    const int e8 = exponent8(largest[i]);
    const float inv = inverse_power(e8);
#pragma unroll
    for (int j = 0; j < JS; j++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][j][4 * q] * inv, acc[i][j][4 * q + 1] * inv, 0, false);
        p = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][j][4 * q + 2] * inv, acc[i][j][4 * q + 3] * inv, p, true);
        *(int *)(st + l32 * PITCH + 32 * j + 8 * q + 4 * hi) = p;
      }
    __builtin_amdgcn_wave_barrier();
    if (hi == 0 && (!SHARED || wn % 2 == 0) && r0 + l32 < rows)
      a.qs[(r0 + l32) * a.qsstride + block] = (uint8_t)(e8 + 127);
#pragma unroll
    for (int k = 0; k < PIECES / 2; k++) {
      const int piece = k * 64 + lane, row = piece / PIECES, col = piece % PIECES * 16;
      if (r0 + row < rows)
        *(u32x4 *)(a.q + (r0 + row) * a.qstride + out0 + col) = *(const u32x4 *)(st + row * PITCH + col);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T, bool EXACT, typename Y, Kind8 KIND>
__global__ __launch_bounds__(T::THREADS, T::FM * T::FN > 8 ? 1 : 2) void k_tile8(Args8 a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % T::WM, wn = wave / T::WM;

  // Each XCD a band of the tiles, in groups of 8 row tiles: neighbours share rows and weights.
  int tiles = gridDim.x, tiles_m = a.tiles_m;
  if constexpr (KIND != PLAIN8) {  // (the launch has room for one more tile an expert than there may be)
    tiles_m = *a.total;
    tiles = tiles_m * a.tiles_n;
    if ((int)blockIdx.x >= tiles) return;
  }
  const int xcd = blockIdx.x & 7, full = tiles >> 3, rest = tiles & 7;
  const int at = xcd * full + min(xcd, rest) + (blockIdx.x >> 3);
  const int group = at / (8 * a.tiles_n), gm = min(8, tiles_m - 8 * group), in_group = at - group * 8 * a.tiles_n;
  const int tile_m = 8 * group + in_group % gm;
  const long n0 = (long)(in_group / gm) * T::TN;
  long m0 = (long)tile_m * T::TM, rows = a.rows, expert = 0;
  if constexpr (KIND != PLAIN8) {
    const ExpertTile t = a.list[tile_m];
    expert = __builtin_amdgcn_readfirstlane(t.expert);
    m0 = __builtin_amdgcn_readfirstlane(t.begin);
    rows = __builtin_amdgcn_readfirstlane(t.end);
  }

  // Where the tile's first row lies, and the others relative to it.
  long oy0 = 0, ox0 = a.row0 + m0, first = ox0;
  if (KIND == PLAIN8 && a.image) {
    const long p = a.row0 + m0, im = p / (a.OH * a.OW), q = p - im * a.OH * a.OW;
    oy0 = q / a.OW;
    ox0 = q - oy0 * a.OW;
    first = (im * a.H + oy0 * a.step) * a.W + ox0 * a.step;
  }
  if constexpr (KIND >= EXPERTS_ACT8) first = 0;
  // Row r of the tile: its pixel after the first one's, and a bit for each
  // tap that falls on the map.
  auto place = [&](int r, int *pixel) {
    *pixel = r;
    if (m0 + r >= rows) return 0;
    if constexpr (KIND >= EXPERTS_ACT8) *pixel = a.order[m0 + r] / a.top;
    if (KIND != PLAIN8 || !a.image) return 1;
    const unsigned x = (unsigned)ox0 + r, down = x / (unsigned)a.OW, ox = x - down * (unsigned)a.OW;
    const unsigned y = (unsigned)oy0 + down, maps = y / (unsigned)a.OH, oy = y - maps * (unsigned)a.OH;
    *pixel = ((int)(maps * (unsigned)a.H) + ((int)oy - (int)oy0) * a.step) * (int)a.W + ((int)ox - (int)ox0) * a.step;
    if (a.taps == 1) return 1;
    const int iy = oy * a.step, ix = ox * a.step;
    const int across = (ix > 0 ? 1 : 0) | 2 | (ix + 1 < a.W ? 4 : 0);
    return (iy > 0 ? across : 0) | across << 3 | (iy + 1 < a.H ? across << 6 : 0);
  };
  int off[T::A_LOADS], mask[T::A_LOADS];
#pragma unroll
  for (int i = 0; i < T::A_LOADS; i++) {
    const int row = (wave + T::WAVES * i) * 8 + (lane >> 3);
    mask[i] = place(row, &off[i]);
    off[i] = off[i] * (int)a.xs + 16 * ((lane & 7) ^ (row >> 1 & 7));
  }
  int soff[T::S_LOADS], smask[T::S_LOADS];
#pragma unroll
  for (int i = 0; i < T::S_LOADS; i++) {
    const int piece = wave + T::WAVES * i;  // (past the scales: into the stage's spare lines)
    smask[i] = piece < T::TM / 64 ? place(piece * 64 + lane, &soff[i]) : -1;
    soff[i] = piece < T::TM / 64 ? soff[i] * (int)a.ss : (piece * 64 + lane - T::TM) * 4;
  }

  // The stream of blocks to load, from this split's first: a tap and a block of
  // its channels, as a uniform offset from where the tile's first row has its
  // first tap.  (One step costs a wave that is alone on its SIMD some 4 cycles an
  // instruction, so a step has few: the taps' offsets are lanes of a register,
  // and nothing asks whether a block is past the last one.  Those are read,
  // SLACK8 panels further on at most, and not multiplied.)
  const int chunks = min(a.taps * a.cb - (int)blockIdx.y * a.kchunks, a.kchunks), c_begin = blockIdx.y * a.kchunks;
  int tap = c_begin / a.cb, ib = c_begin - tap * a.cb;
  const long corner = first - (a.taps == 9 ? a.W + 1 : 0);
  const int t9 = a.taps == 9 ? min(lane, 8) : 0;
  const int tap_pixels = t9 / 3 * (int)a.W + t9 % 3;
  const int tap_bytes = tap_pixels * (int)a.xs, tap_scales = tap_pixels * (int)a.ss;
  int xo, so, vo = 0;
  auto at_tap = [&] {
    xo = __builtin_amdgcn_readlane(tap_bytes, tap) + ib * BLOCK8;
    so = __builtin_amdgcn_readlane(tap_scales, tap) + ib;
  };
  at_tap();
  const int4v xr = uniform_rsrc(a.x + corner * a.xs, 0x7fffff00), sr = uniform_rsrc(a.scales + corner * a.ss, 0x7fffff00);
  const int4v vr = uniform_rsrc(a.ws + ((expert * a.cb + c_begin) * a.npad + n0), 0x7fffff00);
  const uint8_t *w = a.w + ((expert * a.cb + c_begin) * a.npad + n0) * BLOCK8;
  const unsigned wave_lds = __builtin_amdgcn_readfirstlane(lds_addr(lds) + wave * 1024);
  const unsigned wave_lds4 = __builtin_amdgcn_readfirstlane(lds_addr(lds) + wave * 256);
  int woff[T::B_LOADS];
#pragma unroll
  for (int i = 0; i < T::B_LOADS; i++) {
    const int row = (wave + T::WAVES * i) * 8 + (lane >> 3);
    woff[i] = row * BLOCK8 + 16 * ((lane & 7) ^ (row >> 1 & 7));
  }
  // Load I of the block into stage STAGE, by this wave: first its rows, then
  // its weights, then its scales.
  auto load = [&](auto stage, auto I) {
    constexpr int BASE = decltype(stage)::value * T::STAGE, i = decltype(I)::value;
    auto on_map = [&](int off, int mask) {  // or past the end, which reads zeros
      return off | (__builtin_amdgcn_sbfe(~mask, tap, 1) & 0x7fffff00);
    };
    if constexpr (i < T::A_LOADS) {
      dma16_at<BASE + T::WAVES * i * 1024>(xr, wave_lds, on_map(off[i], mask[i]), xo);
    } else if constexpr (i < T::A_LOADS + T::B_LOADS) {
      constexpr int k = i - T::A_LOADS;
      int4v wr = xr;
      wr.x = (int)(long)w;
      wr.y = (int)((long)w >> 32);
      dma16_at<BASE + T::B0 + T::WAVES * k * 1024>(wr, wave_lds, woff[k], 0);
    } else {
      constexpr int k = i - T::A_LOADS - T::B_LOADS, AT = BASE + T::SX0 + T::WAVES * k * 256;
      const bool rows = wave + T::WAVES * k < T::TM / 64;  // (no branch: the products would be moved across it)
      dma1_at<AT>(rows ? sr : vr, wave_lds4, on_map(soff[k], smask[k]), rows ? so : vo);
    }
  };
  auto advance = [&] {
    w += a.npad * BLOCK8;
    vo += (int)a.npad * 4;
    const bool over = ++ib == a.cb;
    tap = over ? tap + 1 : tap;
    ib = over ? 0 : ib;
    at_tap();
  };

  // Half s of a block: 16-byte slots 4 s + 2 hi, + 1 of each row, at those
  // places xor row % 8 (no two of eight neighbouring rows on one bank).
  struct Half {
    int8v x[T::FM], w[T::FN];
  };
  int place16[4];
#pragma unroll
  for (int k = 0; k < 4; k++) place16[k] = l32 * BLOCK8 + 16 * ((4 * (k >> 1) + 2 * hi + (k & 1)) ^ (l32 >> 1 & 7));
  const unsigned char *xp = lds + wm * T::FM * 32 * BLOCK8, *wp = lds + T::B0 + wn * T::FN * 32 * BLOCK8;
  const unsigned char *sp = lds + T::SX0 + (wm * T::FM * 32 + l32) * 4, *vp = lds + T::SW0 + (wn * T::FN * 32 + l32) * 4;
  // Fragment I of half s: the rows' first, then the weights'.
  auto read = [&](Half &h, auto stage, auto s, auto I) {
    constexpr int BASE = decltype(stage)::value * T::STAGE, i = decltype(I)::value, S = decltype(s)::value;
    const unsigned char *p = i < T::FM ? xp + BASE + i * 32 * BLOCK8 : wp + BASE + (i - T::FM) * 32 * BLOCK8;
    const int4v lo = *(const int4v *)(p + place16[2 * S]), up = *(const int4v *)(p + place16[2 * S + 1]);
    const int8v v = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (i < T::FM)
      h.x[i] = v;
    else
      h.w[i - T::FM] = v;
  };
  struct Scales {
    int x[T::FM], w[T::FN];
  };
  auto read_scales = [&](Scales &v, auto stage) {
    constexpr int BASE = decltype(stage)::value * T::STAGE;
#pragma unroll
    for (int i = 0; i < T::FM; i++) v.x[i] = *(const int *)(sp + BASE + i * 128);
#pragma unroll
    for (int j = 0; j < T::FN; j++) v.w[j] = *(const int *)(vp + BASE + j * 128);
  };
  floatx16 acc[T::FM][T::FN] = {};
  constexpr int PRODUCTS = T::FM * T::FN;
  // The products of half a block, beside(k) after each.
  auto multiply = [&](const Half &h, const Scales &v, auto beside) {
    if constexpr (!EXACT) {
      each<PRODUCTS>([&](auto k) {
        constexpr int i = decltype(k)::value / T::FN, j = decltype(k)::value % T::FN;
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(h.w[j], h.x[i], acc[i][j], 0, 0, 0, v.w[j], 0, v.x[i]);
        __builtin_amdgcn_sched_barrier(0);
        beside(k);
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      each<4>([&](auto e) {
        constexpr int E = 2 * decltype(e)::value;
        bf16x8 x[T::FM], w[T::FN];
#pragma unroll
        for (int i = 0; i < T::FM; i++) x[i] = widen8(h.x[i][E], h.x[i][E + 1], scale_power(v.x[i]));
#pragma unroll
        for (int j = 0; j < T::FN; j++) w[j] = widen8(h.w[j][E], h.w[j][E + 1], scale_power(v.w[j]));
        each<PRODUCTS>([&](auto k) {
          constexpr int i = decltype(k)::value / T::FN, j = decltype(k)::value % T::FN;
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], x[i], acc[i][j], 0, 0, 0);
          if constexpr (E == 0) beside(k);
        });
      });
    }
  };

  // Block c's second half is read while its first is multiplied.  Then every
  // wave has read all of it, the next block has landed, and under the second
  // half's products the next one's first half is read and the block S further
  // loaded into this one's place.  (What comes past the last block is not multiplied.)
  if (wave < T::TN / 64)  // the epilogue's biases
    dma_lds4(uniform_rsrc(a.bias + expert * a.npad + n0, (a.npad - n0) * 4), wave_lds4 + T::BIAS0, (wave * 64 + lane) * 4);
  each<T::S>([&](auto stage) {
    each<T::LOADS>([&](auto i) { load(stage, i); });
    advance();
  });
  wait_vm<(T::S - 1) * T::LOADS>();
  lds_barrier();
  constexpr int FRAGS = T::FM + T::FN, EARLY = (PRODUCTS + 1) / 2;  // products among which the fragments are read
  Half h0, h1;
  Scales v[T::S];
  each<FRAGS>([&](auto i) { read(h0, Const<0>{}, Const<0>{}, i); });
  read_scales(v[0], Const<0>{});
  // The products of `now` while half s of stage NEXT is read into `then`, and where `loads`, stage STAGE's next block loaded.
  auto work = [&](const Half &now, const Scales &v, Half &then, auto next, auto s, auto stage, auto loads) {
    multiply(now, v, [&](auto k) {
      constexpr int K = decltype(k)::value, from = share8(K, FRAGS, EARLY), to = share8(K + 1, FRAGS, EARLY);
      each<to - from>([&](auto i) { read(then, next, s, Const<from + decltype(i)::value>{}); });
      if constexpr (decltype(loads)::value) {
        constexpr int first = K * T::LOADS / PRODUCTS, last = (K + 1) * T::LOADS / PRODUCTS;
        each<last - first>([&](auto i) { load(stage, Const<first + decltype(i)::value>{}); });
      }
    });
  };
  auto step = [&](auto stage) {
    constexpr int s = decltype(stage)::value;
    const Const<(s + 1) % T::S> next;
    work(h0, v[s], h1, stage, Const<1>{}, stage, Const<0>{});
    wait_vm<(T::S - 2) * T::LOADS>();
    lds_barrier();
    read_scales(v[next], next);
    work(h1, v[s], h0, next, Const<0>{}, stage, Const<1>{});
    advance();
  };
  int c = 0;
  for (; c + T::S <= chunks; c += T::S) each<T::S>(step);
  each<T::S - 1>([&](auto stage) {
    if (c + decltype(stage)::value < chunks) step(stage);
  });
  wait_vm<0>();
  __syncthreads();  // no load is on its way into LDS, every wave is done with the stages

  if (KIND == PLAIN8 && a.ksplit > 1) {
    ConvArgs split{};
    split.part = a.part;
    split.tile_count = a.tile_count;
    split.ksplit = a.ksplit;
    if (!count_in<T::FM, T::FN, T::THREADS>(split, acc, (int *)lds, tid)) return;
    __syncthreads();
  }

  if constexpr (KIND >= EXPERTS_ACT8) {
    into_rows8<T, KIND == EXPERTS_GATED8>(a, acc, lds, m0, rows, n0, tid);
    return;
  }

  // Each wave 32 of its rows at a time through LDS of its own, for whole lines
  // out: eights of a row's outputs, always the same ones for a lane.
  float *st = (float *)lds + wave * 32 * T::PITCH;
  constexpr int COLS = 32 * T::FN, EIGHTS = COLS / 8, ITEMS = 32 * EIGHTS / 64;
  const long nw = n0 + wn * COLS;
  const int row = lane / EIGHTS, col = lane % EIGHTS * 8;
  float bias[8];
  // Eight floats of LDS, 16-byte aligned.
  auto take = [](const float *p, float *v) {
    const float4v a = *(const float4v *)p, b = *(const float4v *)(p + 4);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = a[k], v[4 + k] = b[k];
  };
  take((const float *)(lds + T::BIAS0) + wn * COLS + col, bias);
  auto stage_rows = [&](const floatx16 (&v)[T::FN]) {
#pragma unroll
    for (int j = 0; j < T::FN; j++)
#pragma unroll
      for (int q = 0; q < 4; q++)
        *(float4v *)(st + l32 * T::PITCH + 32 * j + 8 * q + 4 * hi) =
            float4v{v[j][4 * q], v[j][4 * q + 1], v[j][4 * q + 2], v[j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
  };
  const int many = (int)max(min(a.n - nw - col, 8L), 0L);  // this lane's outputs of an eight
  const bool ragged = nw + COLS > a.n && a.n % 8 != 0;      // (the same for the wave)
  constexpr int STEP = 64 / EIGHTS;                         // rows between its eights
  with_act8(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < T::FM; i++) {
      const long r0 = m0 + (wm * T::FM + i) * 32 + row;
      Y *y = (Y *)a.y + r0 * a.ys + nw + col;
      float old[ITEMS][8];
      if (a.add) {
        const Y *add = (const Y *)a.add + r0 * a.as + nw + col;
#pragma unroll
        for (int e = 0; e < ITEMS; e++) {
          if (r0 + e * STEP >= rows) continue;
          if (many == 0) continue;
          if (!ragged || many == 8)
            load8<Y, true>(add + e * STEP * a.as, 0, 0, old[e]);
          else
            load8<Y, false>(add + e * STEP * a.as, 0, many, old[e]);
        }
      }
      stage_rows(acc[i]);
#pragma unroll
      for (int e = 0; e < ITEMS; e++) {
        if (many == 0 || r0 + e * STEP >= rows) continue;
        float v[8];
        take(st + (row + e * STEP) * T::PITCH + col, v);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += bias[k];
        if (a.add) {
#pragma unroll
          for (int k = 0; k < 8; k++) v[k] += old[e][k];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = act8<decltype(act)::value>(v[k]);
        // (The plan's rows are read again at once: through the caches 8192 tokens, eight of 64 experts each, 1024 -> 1024 in f16
        // 170 -> 161 us with their sums.)
        if (KIND == EXPERTS_ROWS8 && many == 8)
          store8<Y, true>(y + e * STEP * a.ys, 0, 0, v);
        else if (!ragged || many == 8)
          stream8(y + e * STEP * a.ys, v);
        else
          store8<Y, false>(y + e * STEP * a.ys, 0, many, v);
      }
      __builtin_amdgcn_wave_barrier();
    }
  });
}

}  // namespace
}  // namespace ien
