// multiply8.hip -- products of rows in 8 bits with weights in 8 bits, plain
// rows and 3 x 3 convolutions (ien_multiply8), on the scaled 8-bit matrix
// instructions of gfx950:
//   y[r][n] = act(sum over blocks b of 2^(ex[r][b] + ew[b][n])
//                 sum over k in b of qx[r][k] qw[k][n] + bias[n] + add[r][n])
// v_mfma_scale_f32_32x32x64 takes a scale byte a row and 32 values of each
// operand; a block of 128 is two instructions under the same bytes, so the
// scales cost no vector instruction a product.
//
// The 8-bit instructions cut each aligned eight products off towards zero at
// 2^-13 of the power of two of the largest before they add them (measured: of
// 2^16 + v the multiples of 8 in v are left; an operand under 2^-6 counts as
// 2^-6; the eights are then added in f32).  A product under 2^-7 of the largest
// loses bits by that: sums of 64 random products are off by 1.4e-5 of themselves,
// and by all of themselves where large products cancel.  That is no sum in f32, and
// left to a caller who asks for it (`fast`, f16 outputs).  All others take their
// operands as bf16, which holds e4m3 values under scales 3 .. 246 exactly (past
// those it ends: 2^128, 2^-133), and the bf16 instructions (6e-9), at half the rate.  (Rounded to 8 bits again
// after a norm, f16 results off by 1.4e-5 gave a residual block of 64 x 64 x 512
// an error of 4.6e-4 in place of 2.2e-4.)
//
// A workgroup of four waves computes a tile of rows x outputs, a block of 128
// deep at a time through a ring of stages in LDS that buffer loads fill without
// registers; the 3 x 3 taps are the blocks' order, each lane's row at the tap's
// pixel or, off the map, past the buffer's end.  A block takes the 256 x 256
// tile 2.9 us (1.48 PFLOP/s over all CUs; fast 1.45, 2.96), of which the matrix
// pipe is busy in 56 % of the cycles: more than the library's products reach on
// this card (1.32, 2.73), what the other cycles go to was not isolated (it is 12
// bytes a lane short of registers).  Smaller tiles are bound by their way into
// and out of LDS and, a workgroup a CU, by the time a block takes from one barrier
// to the next; they are for what would leave CUs idle.  16384 rows 2048 -> 8192:
// 431 us, fast 245.

#include <algorithm>

#include "eight_bits.h"

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
};

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

template <typename T, bool EXACT, typename Y>
__global__ __launch_bounds__(T::THREADS, T::FM * T::FN > 8 ? 1 : 2) void k_tile8(Args8 a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % T::WM, wn = wave / T::WM;

  // Each XCD a band of the tiles, in groups of 8 row tiles: neighbours share rows and weights.
  const int tiles = gridDim.x, xcd = blockIdx.x & 7, full = tiles >> 3, rest = tiles & 7;
  const int at = xcd * full + min(xcd, rest) + (blockIdx.x >> 3);
  const int group = at / (8 * a.tiles_n), gm = min(8, a.tiles_m - 8 * group), in_group = at - group * 8 * a.tiles_n;
  const long m0 = (long)(8 * group + in_group % gm) * T::TM;
  const long n0 = (long)(in_group / gm) * T::TN;

  // Where the tile's first row lies, and the others relative to it.
  long oy0 = 0, ox0 = a.row0 + m0, first = ox0;
  if (a.image) {
    const long p = a.row0 + m0, im = p / (a.OH * a.OW), q = p - im * a.OH * a.OW;
    oy0 = q / a.OW;
    ox0 = q - oy0 * a.OW;
    first = (im * a.H + oy0 * a.step) * a.W + ox0 * a.step;
  }
  // Row r of the tile: its pixel after the first one's, and a bit for each
  // tap that falls on the map.
  auto place = [&](int r, int *pixel) {
    *pixel = r;
    if (m0 + r >= a.rows) return 0;
    if (!a.image) return 1;
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
  const int4v vr = uniform_rsrc(a.ws + (long)c_begin * a.npad + n0, 0x7fffff00);
  const uint8_t *w = a.w + ((long)c_begin * a.npad + n0) * BLOCK8;
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
    dma_lds4(uniform_rsrc(a.bias + n0, (a.npad - n0) * 4), wave_lds4 + T::BIAS0, (wave * 64 + lane) * 4);
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

  if (a.ksplit > 1) {
    ConvArgs split{};
    split.part = a.part;
    split.tile_count = a.tile_count;
    split.ksplit = a.ksplit;
    if (!count_in<T::FM, T::FN, T::THREADS>(split, acc, (int *)lds, tid)) return;
    __syncthreads();
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
          if (r0 + e * STEP >= a.rows) continue;
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
        if (many == 0 || r0 + e * STEP >= a.rows) continue;
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
        if (!ragged || many == 8)
          stream8(y + e * STEP * a.ys, v);
        else
          store8<Y, false>(y + e * STEP * a.ys, 0, many, v);
      }
      __builtin_amdgcn_wave_barrier();
    }
  });
}

// The tiles a launch chooses among, largest first, and what they were measured
// at: us a block of depth of one tile on a CU alone and among its neighbours,
// with 8-bit and with bf16 instructions, and us a round of tiles for their
// outputs (with a residual to add, where no second workgroup of the CU hides it).
struct Choice8 {
  int tm, tn;
  double alone[2], among[2], out, out_add;
};
constexpr Choice8 CHOICES8[] = {{256, 256, {1.45, 2.9}, {1.45, 2.9}, 8.0, 25.0},
                                {128, 128, {0.65, 0.90}, {0.50, 0.72}, 3.0, 3.8},
                                {64, 128, {0.38, 0.68}, {0.27, 0.46}, 1.7, 2.8},
                                {64, 64, {0.38, 0.60}, {0.22, 0.34}, 1.2, 2.0}};

template <typename T>
void launch(ien_ctx *ctx, Args8 &a) {
  const dim3 grid((unsigned)(a.tiles_m * a.tiles_n), (unsigned)a.ksplit);
  if (a.f32)
    hipLaunchKernelGGL((k_tile8<T, true, float>), grid, dim3(T::THREADS), 0, ctx->stream, a);
  else if (a.exact)
    hipLaunchKernelGGL((k_tile8<T, true, _Float16>), grid, dim3(T::THREADS), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL((k_tile8<T, false, _Float16>), grid, dim3(T::THREADS), 0, ctx->stream, a);
}

void run_part(ien_ctx *ctx, Args8 &a, int tile, int ksplit) {
  const int chunks = a.taps * a.cb;
  const Choice8 &c = CHOICES8[tile];
  a.tiles_m = (int)((a.rows + c.tm - 1) / c.tm);
  a.tiles_n = (int)((a.n + c.tn - 1) / c.tn);
  a.ksplit = ksplit;
  a.kchunks = (chunks + ksplit - 1) / ksplit;
  a.part = ctx->splitk;
  a.tile_count = (int *)(ctx->splitk + ctx->splitk_floats);
  const bool shared = (long)a.tiles_m * a.tiles_n * a.ksplit > ctx->cus;
  switch (tile) {
    case 0: launch<Tile8<4, 4, 2, 2, 2>>(ctx, a); break;
    case 1:
      // Twice the waves: fast sums, for the residuals' loads (4096 rows 384 -> 1536 11.3 -> 9.9 us, 3x3 256x384 128 ->
      // 128 27.2 -> 23.6; without a residual 16384 rows 2048 -> 8192 293 -> 296).  Exact ones, where a CU has one
      // workgroup (2048 rows 8192 -> 2048 68.3 -> 63.8, with a residual 1024 rows 4096 -> 4096 38.9 -> 36.6);
      // among others they lose (3x3 256x384 256 -> 256 97 -> 115, with a residual 102 -> 125).
      (a.exact ? !shared : a.add != nullptr) ? launch<Tile8<1, 2, 4, 2, 2>>(ctx, a) : launch<Tile8<2, 2, 2, 2, 2>>(ctx, a);
      break;
    case 2:
      // Three workgroups a CU with two stages, where there are as many: 4096 rows 384 -> 1536 11.0 -> 10.0 us (fast 9.4 ->
      // 7.9).  One a CU wants three: 3x3 64x64 512 -> 512 with a residual 26.8 -> 25.0 (fast 21.5 -> 17.2).
      shared ? launch<Tile8<1, 2, 2, 2, 2>>(ctx, a) : launch<Tile8<1, 2, 2, 2, 3>>(ctx, a);
      break;
    default: launch<Tile8<1, 1, 2, 2, 4>>(ctx, a); break;
  }
}

void run_tiles(ien_ctx *ctx, const Args8 &a) {
  const int plan = multiply8_choice(ctx->cus, (long)ctx->splitk_floats, a.rows, a.n, a.taps * a.cb, a.exact, a.add);
  const long part = multiply8_part(plan / 64, a.n);
  for (long r = 0; r < a.rows; r += part) {  // (one turn but for some 10^10 outputs)
    Args8 p = a;
    p.row0 += r;
    p.rows = std::min(part, a.rows - r);
    p.y = (uint8_t *)a.y + r * a.ys * (a.f32 ? 4 : 2);
    if (a.add) p.add = (const uint8_t *)a.add + r * a.as * (a.f32 ? 4 : 2);
    run_part(ctx, p, plan / 64, plan % 64);
  }
}

}  // namespace

// 2^21 tiles, which at 512 lanes are 2^30: a launch counts its lanes in 32 bits.
long multiply8_part(int tile, long n) {
  const Choice8 &c = CHOICES8[tile];
  return std::max((1L << 21) / ((n + c.tn - 1) / c.tn), 1L) * c.tm;
}

// The tile (times 64) and in how many splits of the depth: by the estimated
// time.  Few tiles leave CUs idle, which splits fill for a pass through device
// memory and about 5 us.
int multiply8_choice(int cus, long workspace, long rows, long n, int chunks, bool exact, bool add) {
  int best = -1;
  double best_us = 1e30;
  for (int t = 0; t < 4; t++) {
    const Choice8 &c = CHOICES8[t];
    const long tiles = ((rows + c.tm - 1) / c.tm) * ((n + c.tn - 1) / c.tn);
    for (int ks = 1; ks <= 16 && ks <= chunks; ks++) {
      if (ks > 1 && (tiles * ks > 2 * cus || tiles > ien_ctx::SPLITK_TILES || tiles * ks * c.tm * c.tn > workspace)) break;
      const int deep = (chunks + ks - 1) / ks;
      if ((chunks + deep - 1) / deep != ks) continue;
      const long rounds = (tiles * ks + cus - 1) / cus;
      double us = (rounds == 1 ? c.alone[exact] : rounds * c.among[exact]) * deep + rounds * (add ? c.out_add : c.out);
      if (ks > 1) us += 5.0 + 3e-6 * (double)(tiles * ks) * c.tm * c.tn;
      if (us < best_us) best_us = us, best = 64 * t + ks;
    }
  }
  return best;
}

}  // namespace ien

using namespace ien;

extern "C" {

ien_status ien_multiply8(ien_ctx *ctx, const ien_input8 *in, size_t row0, size_t rows, const ien_matrix8 *w,
                         const ien_output *out, ien_act act, const void *d_add, size_t add_stride) {
  IEN_CHECK(ctx && in && w && w->d_w && out, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(act8_known(act), IEN_ERR_INPUT, "multiply8 takes no activation %d", (int)act);
  IEN_CHECK(out->type == IEN_OUT_F16 || out->type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)out->type);
  IEN_CHECK(out->layout == IEN_LAYOUT_NHWC, IEN_ERR_INPUT, "multiply8 writes NHWC rows");
  Args8 a{};
  a.taps = (int)w->taps;
  a.cb = w->cb;
  a.step = 1;
  if (in->kind == IEN_INPUT_ROWS) {
    IEN_CHECK(w->taps == 1, IEN_ERR_INPUT, "%zu taps on rows", w->taps);
    IEN_CHECK(row0 < (1ull << 40) && rows < (1ull << 40), IEN_ERR_INPUT, "rows %zu..%zu", row0, row0 + rows);
    a.images = a.H = a.OH = 1;
    a.W = a.OW = (long)(row0 + rows);
  } else {
    IEN_CHECK(in->kind == IEN_INPUT_IMAGE, IEN_ERR_INPUT, "input kind %d", (int)in->kind);
    IEN_CHECK(in->step == 1 || in->step == 2, IEN_ERR_INPUT, "step %zu", in->step);
    IEN_CHECK(in->images < (1u << 20) && in->height < (1u << 20) && in->width < (1u << 20), IEN_ERR_INPUT,
              "%zu maps of %zu x %zu", in->images, in->height, in->width);
    a.step = (int)in->step;
    a.images = (long)in->images;
    a.H = (long)in->height;
    a.W = (long)in->width;
    a.OH = (a.H + a.step - 1) / a.step;
    a.OW = (a.W + a.step - 1) / a.step;
    const size_t pixels = (size_t)(a.images * a.OH * a.OW);
    IEN_CHECK(row0 <= pixels && rows <= pixels - row0, IEN_ERR_INPUT, "rows %zu..%zu past %zu pixels", row0,
              row0 + rows, pixels);
  }
  if (rows == 0) return IEN_OK;
  const ien_status s = check_rows8(&in->map, w->c, "multiply8");
  if (s != IEN_OK) return s;
  IEN_CHECK(out->data && out->stride >= w->n && (!d_add || add_stride >= w->n), IEN_ERR_INPUT,
            "no output, or rows %zu and %zu apart for n = %zu", out->stride, add_stride, w->n);
  a.x = in->map.data;
  a.xs = (long)in->map.stride;
  a.scales = in->map.scales;
  a.ss = (long)in->map.scale_stride;
  a.row0 = (long)row0;
  a.rows = (long)rows;
  a.w = w->d_w;
  a.ws = w->d_scales;
  a.bias = w->d_bias;
  a.n = (long)w->n;
  a.npad = w->npad;
  a.y = out->data;
  a.ys = (long)out->stride;
  a.f32 = out->type == IEN_OUT_F32;
  a.exact = a.f32 || !in->fast;
  a.act = act;
  a.add = d_add;
  a.as = (long)add_stride;
  a.image = in->kind == IEN_INPUT_IMAGE;
  // A tile addresses its rows' values by 31-bit offsets from its first one's.
  IEN_CHECK(in->map.stride < (1u << 20) && in->map.scale_stride < (1u << 20) &&
                (!a.image || (in->width + 256) * std::max(in->map.stride, in->map.scale_stride) < (1u << 27)) &&
                w->taps * w->cb * w->npad < (1l << 28),
            IEN_ERR_INPUT, "rows in 8 bits %zu and %zu bytes apart, %ld to a line of a map, or too many weights", in->map.stride,
            in->map.scale_stride, a.W);
  run_tiles(ctx, a);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

}  // extern "C"
