// experts_out8.hip -- the experts' second product and each token's weighted sum
// of it (ien_experts_out8): the rows of the plan times their experts' weights in
// ien_multiply8's tiles (tile8.h), then, a token after another, its pairs' rows
// by their weights onto the residual.  The sum is a pass of its own, so that it
// takes the slots in order: what arrives first decides nothing.

#include <algorithm>
#include <type_traits>

#include "few8.h"

namespace ien {
namespace {

template <typename T>
bool launch(ien_ctx *ctx, Args8 &a, const ien_routes *r, const PlanLayout &p, int size) {
  a.tiles_n = (int)((a.n + T::TN - 1) / T::TN);
  a.list = (const ExpertTile *)(r->d_plan + p.tiles[size]);
  a.total = r->d_plan + p.totals + size;
  if (!launches(p.most[size], a.tiles_n, T::THREADS)) return false;
  const dim3 grid((unsigned)(p.most[size] * a.tiles_n));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(T::THREADS), 0, ctx->stream, a); };
  if (a.exact)
    a.f32 ? go(k_tile8<T, true, float, EXPERTS_ROWS8>) : go(k_tile8<T, true, _Float16, EXPERTS_ROWS8>);
  else
    a.f32 ? go(k_tile8<T, false, float, EXPERTS_ROWS8>) : go(k_tile8<T, false, _Float16, EXPERTS_ROWS8>);
  return true;
}

template <int WN, int WK>
bool few(ien_ctx *ctx, Args8 &a, const ien_routes *r, const PlanLayout &p) {
  return a.f32 ? launch_few<EXPERTS_ROWS8, float, WN, WK>(ctx, a, r, p)
               : launch_few<EXPERTS_ROWS8, _Float16, WN, WK>(ctx, a, r, p);
}

struct CombineArgs {
  const void *parts;
  long pitch;
  const int *place;
  const float *weight;
  const void *add;  // of the result's type
  long as;
  const void *branch;
  long bs;
  int branch_f32;
  void *y;
  long ys;
  long tokens, n;
  int top;
};

// A lane eight outputs of a token (Y) from rows of parts (P), which are whole eights.  All
// sums are in f32: an f16 result of f32 parts is rounded once.  Memory bounds it: 16384 x
// 1024, four experts each, with a residual of two addends 66 us of f32 parts, 5.5 TB/s, and
// 41 of f16 ones.  (With their product 8192 tokens, eight experts each, 1024 -> 1024 225 and
// 165 us: where products are known to be within f16, and its rounding does, they may be.)
template <typename Y, typename P>
__global__ __launch_bounds__(256) void k_combine(CombineArgs a) {
  const long eights = (a.n + 7) / 8, total = a.tokens * eights;
  for (long item = (long)blockIdx.x * 256 + threadIdx.x; item < total; item += (long)gridDim.x * 256) {
    const long t = item / eights, at = (item - t * eights) * 8;
    const bool whole = at + 8 <= a.n;
    float v[8] = {};
    for (int k = 0; k < a.top; k++) {
      const int place = a.place[t * a.top + k];
      if (place < 0) continue;
      const float w = a.weight[t * a.top + k];
      float part[8];
      load8<P, true>((const P *)a.parts + place * a.pitch, at, 0, part);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = fmaf(w, part[i], v[i]);
    }
    if (a.add || a.branch) {
      float old[8] = {}, branch[8] = {};
      auto load = [&](auto *row, float *v) {
        typedef std::remove_cv_t<std::remove_pointer_t<decltype(row)>> T;
        whole ? load8<T, true>(row, at, 0, v) : load8<T, false>(row, at, a.n, v);
      };
      if (a.add) load((const Y *)a.add + t * a.as, old);
      if (a.branch) a.branch_f32 ? load((const float *)a.branch + t * a.bs, branch) : load((const _Float16 *)a.branch + t * a.bs, branch);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += old[i] + branch[i];
    }
    Y *y = (Y *)a.y + t * a.ys;
    if (whole)
      stream8(y + at, v);
    else
      store8<Y, false>(y, at, a.n, v);
  }
}

}  // namespace

// The size of tile (TILE_ROWS), 0 and 3 for few rows an expert: waves that read the
// weights straight into registers, two shares of the depth beside each other, or four
// where a share then has four blocks at least (us, f16 products, with the sum's pass; 2048 -> 1024: one
// row of 8 experts 9.4, two shares 11.6, tiles of 64 rows 18.1; 1024 -> 1024: two rows of 56
// experts 15.9, four shares 23.8, tiles 18.2; four rows 19.4 and 19.0).  Else two
// workgroups a CU of 128 x 128 outputs or three of 64 x 128 (rows an expert 128: 39.5 and
// 35.1, 512: 21.3 and 21.3, 1024: 34.9 and 41.8, 2048: 287 and 316).
int experts_out_choice(long pairs, long experts, int chunks) {
  const long mean = pairs / std::min(pairs, experts);
  if (mean < 3) return chunks >= 16 ? 3 : 0;
  return mean >= 400 ? 2 : 1;
}

}  // namespace ien

using namespace ien;

extern "C" {

size_t ien_experts_parts(const ien_routes *routes, const ien_experts8 *w) {
  if (!w || check_routes(routes, "experts_parts") != IEN_OK) return 0;
  return routes->tokens * routes->top * ((w->n + 7) / 8 * 8);
}

ien_status ien_experts_out8(ien_ctx *ctx, const ien_rows8 *h, const ien_routes *routes, const ien_experts8 *w,
                            int fast, void *d_parts, const void *d_add, size_t add_stride, const ien_output *out) {
  IEN_CHECK(out, IEN_ERR_INPUT, "null argument");
  return ien_experts_out8_ex(ctx, h, routes, w, fast, d_parts, out->type, d_add, add_stride, nullptr, out->type, 0, out);
}

ien_status ien_experts_out8_ex(ien_ctx *ctx, const ien_rows8 *h, const ien_routes *routes, const ien_experts8 *w,
                               int fast, void *d_parts, ien_out_type parts_type, const void *d_add, size_t add_stride,
                               const void *d_branch, ien_out_type branch_type, size_t branch_stride,
                               const ien_output *out) {
  IEN_CHECK(ctx && w && w->d_w && out, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(!w->gated, IEN_ERR_INPUT, "experts_out8 takes no gated weights");
  IEN_CHECK((out->type == IEN_OUT_F16 || out->type == IEN_OUT_F32) && (parts_type == IEN_OUT_F32 || parts_type == out->type) &&
                (!d_branch || branch_type == IEN_OUT_F16 || branch_type == IEN_OUT_F32),
            IEN_ERR_INPUT, "type %d from products of type %d, with a branch of type %d", (int)out->type, (int)parts_type,
            (int)branch_type);
  IEN_CHECK(out->layout == IEN_LAYOUT_NHWC, IEN_ERR_INPUT, "experts_out8 writes NHWC rows");
  ien_status s = check_routes(routes, "experts_out8");
  if (s != IEN_OK) return s;
  IEN_CHECK(routes->experts == w->experts, IEN_ERR_INPUT, "routes to %zu experts of %zu", routes->experts, w->experts);
  if (routes->tokens == 0) return IEN_OK;
  s = check_rows8(h, w->c, "experts_out8");
  if (s != IEN_OK) return s;
  IEN_CHECK(out->data && out->stride >= w->n && (!d_add || add_stride >= w->n) && (!d_branch || branch_stride >= w->n),
            IEN_ERR_INPUT, "no output, or rows %zu, %zu and %zu apart for n = %zu", out->stride, add_stride, branch_stride,
            w->n);
  IEN_CHECK(d_parts && ((uintptr_t)d_parts & 15) == 0, IEN_ERR_INPUT, "experts_out8: no parts, or unaligned");
  IEN_CHECK(h->stride < (1u << 20) && h->scale_stride < (1u << 20), IEN_ERR_INPUT,
            "experts_out8: rows in 8 bits %zu and %zu bytes apart", h->stride, h->scale_stride);
  const PlanLayout p = plan_layout(routes->tokens, routes->experts, routes->top);
  Args8 a{};
  a.x = h->data;
  a.xs = (long)h->stride;
  a.scales = h->scales;
  a.ss = (long)h->scale_stride;
  a.taps = 1;
  a.step = 1;
  a.images = a.H = a.OH = 1;
  a.cb = w->cb;
  a.w = w->d_w;
  a.ws = w->d_scales;
  a.bias = w->d_bias;
  a.n = (long)w->n;
  a.npad = w->npad;
  a.y = d_parts;
  a.ys = (long)((w->n + 7) / 8 * 8);
  a.f32 = parts_type == IEN_OUT_F32;
  a.exact = out->type == IEN_OUT_F32 || !fast;
  a.act = IEN_ACT_NONE;
  a.ksplit = 1;
  a.kchunks = w->cb;
  const long pairs = (long)(routes->tokens * routes->top);
  bool done = false;
  switch (experts_out_choice(pairs, (long)routes->experts, a.cb)) {
    case 0: done = few<4, 2>(ctx, a, routes, p); break;
    case 1: done = launch<Tile8<1, 2, 2, 2, 2>>(ctx, a, routes, p, 1); break;
    case 2: done = launch<Tile8<2, 2, 2, 2, 2>>(ctx, a, routes, p, 2); break;
    default: done = few<2, 4>(ctx, a, routes, p); break;
  }
  IEN_CHECK(done, IEN_ERR_INPUT, "experts_out8: %ld pairs by %ld columns are too many tiles", pairs, a.n);
  IEN_HIP(hipGetLastError());
  CombineArgs c{d_parts, a.ys, routes->d_plan + p.place, routes->d_weight, d_add, (long)add_stride, d_branch,
                (long)branch_stride, branch_type == IEN_OUT_F32, out->data, (long)out->stride, (long)routes->tokens, a.n,
                (int)routes->top};
  const long items = c.tokens * ((c.n + 7) / 8);
  const dim3 grid((unsigned)std::min((items + 255) / 256, 1L << 20));
  auto combine = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, c); };
  if (out->type == IEN_OUT_F32)
    combine(k_combine<float, float>);
  else
    a.f32 ? combine(k_combine<_Float16, float>) : combine(k_combine<_Float16, _Float16>);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

}  // extern "C"
