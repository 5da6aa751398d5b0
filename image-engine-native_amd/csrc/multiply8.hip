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

#include "tile8.h"

namespace ien {
namespace {

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
    hipLaunchKernelGGL((k_tile8<T, true, float, PLAIN8>), grid, dim3(T::THREADS), 0, ctx->stream, a);
  else if (a.exact)
    hipLaunchKernelGGL((k_tile8<T, true, _Float16, PLAIN8>), grid, dim3(T::THREADS), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL((k_tile8<T, false, _Float16, PLAIN8>), grid, dim3(T::THREADS), 0, ctx->stream, a);
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
