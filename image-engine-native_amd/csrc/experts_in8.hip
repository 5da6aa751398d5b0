// experts_in8.hip -- the experts' first product (ien_experts_in8): the rows of
// each expert's tokens, gathered by the plan, times its weights, with biases, an
// activation or a gate, and rounding to 8 bits in the epilogue.  Tiles are
// ien_multiply8's (tile8.h): a tile is up to 64, 128 or 256 pairs of one expert.

#include <algorithm>
#include <cmath>

#include "few8.h"

namespace ien {
namespace {

template <typename T, bool EXACT, Kind8 KIND>
bool launch_sums(ien_ctx *ctx, Args8 &a, const ien_routes *r, const PlanLayout &p, int size) {
  a.tiles_n = (int)((a.npad + T::TN - 1) / T::TN);
  a.list = (const ExpertTile *)(r->d_plan + p.tiles[size]);
  a.total = r->d_plan + p.totals + size;
  if (!launches(p.most[size], a.tiles_n, T::THREADS)) return false;
  const dim3 grid((unsigned)(p.most[size] * a.tiles_n));
  hipLaunchKernelGGL((k_tile8<T, EXACT, _Float16, KIND>), grid, dim3(T::THREADS), 0, ctx->stream, a);
  return true;
}
template <typename T, Kind8 KIND>
bool launch(ien_ctx *ctx, Args8 &a, const ien_routes *r, const PlanLayout &p, int size) {
  return a.exact ? launch_sums<T, true, KIND>(ctx, a, r, p, size) : launch_sums<T, false, KIND>(ctx, a, r, p, size);
}

}  // namespace

// The size of tile (TILE_ROWS) for that many pairs, columns in whole 128s and blocks
// of depth.  Where an expert has few rows its weights are what is read, and waves that
// read them straight into registers beat a tile's stages: gated, four rows an expert
// 26.8 us against 28.3, eight 34.1 against 29.4 (1024 -> 2 x 1024, 64 experts); plain,
// one row 8.0 against 9.4, two 16.3 against 14.9.
// Plain tiles: two workgroups a CU of 128 x 128 outputs or three of 64 x 128, which
// take 1.1 times as long a row but leave fewer idle (us, rows an expert 128: 40.2 and
// 31.8, 512: 26.3 and 25.2, 1024: 42.0 and 43.4, 2048: 333 and 365).
// Gated ones (2: with the coarser sums) are 256 columns wide, a workgroup a CU: by the
// rounds of workgroups and what a round was measured at, a block and at its end.
int experts_in_choice(int cus, long pairs, long experts, long npad, int chunks, int gated) {
  const long active = std::min(pairs, experts), mean = pairs / active;
  if (mean <= (gated ? 4 : 1)) return 0;
  if (!gated) return mean >= 640 ? 2 : 1;
  constexpr double BLOCK_US[2][3] = {{0.85, 1.65, 2.95}, {0.54, 1.18, 1.48}};
  constexpr double END_US[2][3] = {{4.5, 4.3, 6.3}, {4.2, 4.0, 9.5}};
  int best = 1;
  double best_us = 1e30;
  for (int size = 1; size < TILE_SIZES; size++) {
    // An expert's last tile is part of one, half of it on an average, and more where few tiles are an expert's (loads differ).
    const double rows = TILE_ROWS[size], part = 0.5 + 0.1 * std::min(1.0, rows / (double)mean);
    const double tiles = ((double)pairs / rows + part * (double)active) * (double)((npad + 255) / 256);
    const double us = std::ceil(tiles / cus) * (BLOCK_US[gated - 1][size - 1] * chunks + END_US[gated - 1][size - 1]);
    if (us < best_us) best_us = us, best = size;
  }
  return best;
}

}  // namespace ien

using namespace ien;

extern "C" ien_status ien_experts_in8(ien_ctx *ctx, const ien_rows8 *x, const ien_routes *routes,
                                      const ien_experts8 *w, ien_act act, int fast, const ien_rows8 *out) {
  IEN_CHECK(ctx && w && w->d_w, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(act8_known(act), IEN_ERR_INPUT, "experts_in8 takes no activation %d", (int)act);
  ien_status s = check_routes(routes, "experts_in8");
  if (s != IEN_OK) return s;
  IEN_CHECK(routes->experts == w->experts, IEN_ERR_INPUT, "routes to %zu experts of %zu", routes->experts, w->experts);
  if (routes->tokens == 0) return IEN_OK;
  s = check_rows8(x, w->c, "experts_in8");
  if (s != IEN_OK) return s;
  s = check_rows8(out, w->n, "experts_in8");
  if (s != IEN_OK) return s;
  IEN_CHECK(x->stride < (1u << 20) && x->scale_stride < (1u << 20) && out->stride < (1u << 20) &&
                out->scale_stride < (1u << 20) && routes->tokens * std::max(x->stride, x->scale_stride) < 0x7fffff00,
            IEN_ERR_INPUT, "experts_in8: %zu rows %zu and %zu bytes apart, results %zu and %zu", routes->tokens,
            x->stride, x->scale_stride, out->stride, out->scale_stride);
  const PlanLayout p = plan_layout(routes->tokens, routes->experts, routes->top);
  Args8 a{};
  a.x = x->data;
  a.xs = (long)x->stride;
  a.scales = x->scales;
  a.ss = (long)x->scale_stride;
  a.taps = 1;
  a.step = 1;
  a.images = a.H = a.OH = 1;
  a.cb = w->cb;
  a.w = w->d_w;
  a.ws = w->d_scales;
  a.bias = w->d_bias;
  a.n = (long)w->n;
  a.npad = w->npad;
  a.exact = !fast;
  a.act = act;
  a.ksplit = 1;
  a.kchunks = w->cb;
  a.order = routes->d_plan + p.order;
  a.top = (int)routes->top;
  a.q = out->data;
  a.qstride = (long)out->stride;
  a.qs = out->scales;
  a.qsstride = (long)out->scale_stride;
  const long pairs = (long)(routes->tokens * routes->top);
  bool done = false;
  switch (experts_in_choice(ctx->cus, pairs, (long)routes->experts, a.npad, a.cb, w->gated ? 1 + !a.exact : 0)) {
    case 0:
      done = w->gated ? launch_few<EXPERTS_GATED8, float, 8, 1>(ctx, a, routes, p)
                      : launch_few<EXPERTS_ACT8, float, 8, 1>(ctx, a, routes, p);
      break;
    case 1:
      done = w->gated ? launch<Tile8<1, 4, 2, 2, 3>, EXPERTS_GATED8>(ctx, a, routes, p, 1)
                      : launch<Tile8<1, 2, 2, 2, 2>, EXPERTS_ACT8>(ctx, a, routes, p, 1);
      break;
    case 2:
      done = w->gated ? launch<Tile8<1, 4, 4, 2, 2>, EXPERTS_GATED8>(ctx, a, routes, p, 2)
                      : launch<Tile8<2, 2, 2, 2, 2>, EXPERTS_ACT8>(ctx, a, routes, p, 2);
      break;
    default:
      // Eight waves widen operands beside the others' products (509 us, four waves 705, 16384 tokens, four of 32 experts
      // each, 1024 -> 2 x 2048); there is nothing to widen for the 8-bit instructions, whose operands eight waves have no
      // registers for (1452 us, four waves 362).
      done = a.exact ? launch_sums<Tile8<2, 4, 4, 2, 2>, true, EXPERTS_GATED8>(ctx, a, routes, p, 3)
                     : launch_sums<Tile8<4, 4, 2, 2, 2>, false, EXPERTS_GATED8>(ctx, a, routes, p, 3);
      break;
  }
  IEN_CHECK(done, IEN_ERR_INPUT, "experts_in8: %ld pairs by %ld columns are too many tiles", pairs, a.npad);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}
