// route.hip -- each token's experts from a router's logits, and the pairs of
// tokens and experts in the order of the experts (ien_route, ien_routes_plan).
//
// Choosing.  16 lanes hold a token's scores (64 where there are more than 256
// experts) and find the largest choice among them, top times.  Choices are
// compared in f64: two that differ by less than a step of f32 are still told
// apart, and the order of the sums decides nothing.
//
// Planning is a counting sort that keeps the order of equal experts and adds
// nothing atomically across workgroups, so it is the same every time: counts of
// each chunk of the pairs, the chunks' sums for each expert, then every pair's
// place, a wave taking its part of the chunk 64 pairs at a time (a pair's rank
// among them is the number of lanes before it with its expert).  Plans of one
// chunk take one launch.

#include <algorithm>

#include "experts.h"

namespace ien {

ien_status check_routes(const ien_routes *r, const char *what) {
  IEN_CHECK(r, IEN_ERR_INPUT, "%s: no routes", what);
  IEN_CHECK(r->experts >= 1 && r->experts <= MAX_EXPERTS && r->top >= 1 && r->top <= MAX_TOP && r->top <= r->experts &&
                r->tokens <= MAX_PAIRS / r->top,
            IEN_ERR_INPUT, "%s: %zu tokens, %zu of %zu experts", what, r->tokens, r->top, r->experts);
  if (r->tokens == 0) return IEN_OK;
  IEN_CHECK(r->d_index && r->d_weight && r->d_plan && ((uintptr_t)r->d_plan & 15) == 0 &&
                (((uintptr_t)r->d_index | (uintptr_t)r->d_weight) & 3) == 0,
            IEN_ERR_INPUT, "%s: routes without an index, weights or a plan, or unaligned", what);
  return IEN_OK;
}

namespace {

struct RouteArgs {
  const void *logits;
  long stride, tokens;
  int experts, top;
  const float *bias;
  int softmax, groups, kept, group_top, renormalise;
  float scale;
  int *index;
  float *weight;
};

// (a, i) before (b, j): the larger choice, of equal ones the lower index.
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

// L lanes a token, V experts a lane: expert l + L i.
template <typename X, int L, int V>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
  constexpr int TOKENS = 256 / L;
  extern __shared__ double shared[];  // grouped: [token][experts] choices, then [token][groups] ranks
  const int lane = threadIdx.x % L, slot = threadIdx.x / L, experts = a.experts;
  const long first = (long)blockIdx.x * TOKENS, t = min(first + slot, a.tokens - 1);
  const bool some = first + slot < a.tokens;
  const double none = -__builtin_inf();
  double s[V], c[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + L * i;
    s[i] = e < experts ? (double)((const X *)a.logits)[t * a.stride + e] : none;
    if (!(s[i] > none)) s[i] = none;  // (NaN too)
    c[i] = s[i];
  }
  if (a.softmax) {
    double m = none;
#pragma unroll
    for (int i = 0; i < V; i++) m = fmax(m, s[i]);
#pragma unroll
    for (int k = 1; k < L; k *= 2) m = fmax(m, __shfl_xor(m, k));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      s[i] = s[i] == m ? 1.0 : exp(s[i] - m);  // (infinite ones share all; closed ones are 0)
      if (c[i] == none) s[i] = 0.0;
      sum += s[i];
    }
#pragma unroll
    for (int k = 1; k < L; k *= 2) sum += __shfl_xor(sum, k);
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = 1.0 / (1.0 + exp(-s[i]));
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + L * i;
    const float b = a.bias && e < experts ? a.bias[e] : 0.0f;
    c[i] = c[i] == none || !(b > -__builtin_inff()) ? none : s[i] + (double)b;
  }
  if (a.kept < a.groups) {
    double *choices = shared + slot * experts, *ranks = shared + TOKENS * experts + slot * a.groups;
    const int per = experts / a.groups;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (lane + L * i < experts) choices[lane + L * i] = c[i];
    __syncthreads();
    for (int g = lane; g < a.groups; g += L) {
      double best = none, next = none;
      for (int e = g * per; e < (g + 1) * per; e++) {
        const double v = choices[e];
        next = fmax(next, fmin(best, v));
        best = fmax(best, v);
      }
      ranks[g] = a.group_top == 2 && next > none ? best + next : best;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int e = lane + L * i;
      if (e >= experts) continue;
      const int mine = e / per;
      const double rank = ranks[mine];
      int ahead = 0;
      for (int g = 0; g < a.groups; g++) ahead += before(ranks[g], g, rank, mine);
      if (ahead >= a.kept) c[i] = none;
    }
  }
  // Slot k's expert and score stay with lane k.
  int chosen = -1;
  double score = 0.0, total = 0.0;
  for (int k = 0; k < a.top; k++) {
    double best = none, its = 0.0;
    int at = 1 << 30;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (c[i] > best) best = c[i], at = lane + L * i, its = s[i];
#pragma unroll
    for (int m = 1; m < L; m *= 2) {
      const double other = __shfl_xor(best, m), score_of = __shfl_xor(its, m);
      const int there = __shfl_xor(at, m);
      if (before(other, there, best, at)) best = other, at = there, its = score_of;
    }
#pragma unroll
    for (int i = 0; i < V; i++)
      if (lane + L * i == at) c[i] = none;
    total += its;
    if (lane == k && best > none) chosen = at, score = its;
  }
  if (some && lane < a.top) {
    a.index[t * a.top + lane] = chosen;
    const double w = !a.renormalise ? score : total > 0.0 ? score / total : 0.0;
    a.weight[t * a.top + lane] = (float)(w * (double)a.scale);
  }
}

struct PlanArgs {
  const int *index;
  int *plan;
  long pairs;
  int experts;
  PlanLayout at;
};

constexpr int WAVES = 4;

__device__ __forceinline__ int expert_of(const PlanArgs &a, long pair) {
  const int e = a.index[pair];
  return (unsigned)e < (unsigned)a.experts ? e : a.experts;
}

// Exclusive sums of n (at most 1025) counts in LDS, in place, by 256 threads;
// every thread gets the sum of all.
__device__ int scan_counts(int *v, int n, int *work) {
  constexpr int EACH = (MAX_EXPERTS + 1 + 255) / 256;
  int mine[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int at = threadIdx.x * EACH + i;
    mine[i] = at < n ? v[at] : 0;
    sum += mine[i];
  }
  int before = sum;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const int o = __shfl_up(before, m);
    if ((int)(threadIdx.x & 63) >= m) before += o;
  }
  if ((threadIdx.x & 63) == 63) work[threadIdx.x / 64] = before;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    if (w < (int)threadIdx.x / 64) base += work[w];
    all += work[w];
  }
  int run = base + before - sum;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int at = threadIdx.x * EACH + i;
    if (at < n) v[at] = run;
    run += mine[i];
  }
  __syncthreads();
  return all;
}

// Offsets, and the tiles of each size, from the counts of experts + 1 bins in LDS
// (which become the offsets).
__device__ void lay_out(const PlanArgs &a, int *counts, int *firsts, int *work) {
  for (int s = 0; s < TILE_SIZES; s++) {
    for (int e = threadIdx.x; e < a.experts; e += 256) firsts[e] = (counts[e] + TILE_ROWS[s] - 1) / TILE_ROWS[s];
    __syncthreads();
    const int all = scan_counts(firsts, a.experts, work);
    for (int e = threadIdx.x; e < a.experts; e += 256) a.plan[a.at.firsts + (long)s * a.experts + e] = firsts[e];
    if (threadIdx.x == 0) a.plan[a.at.totals + s] = all;
    __syncthreads();
  }
  scan_counts(counts, a.experts + 1, work);
  for (int e = threadIdx.x; e <= a.experts; e += 256) a.plan[a.at.offsets + e] = counts[e];
  __syncthreads();
}

// Counts of the chunk's pairs by expert, a wave its part: [wave][bin] in LDS.
__device__ void count_chunk(const PlanArgs &a, int *bins, long begin, long end) {
  const int n = a.experts + 1, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < WAVES * n; i += 256) bins[i] = 0;
  __syncthreads();
  const long part = a.at.chunk / WAVES, from = begin + wave * part, to = min(from + part, end);
  for (long p = from + lane; p < to; p += 64) atomicAdd(bins + wave * n + expert_of(a, p), 1);
  __syncthreads();
}

__global__ __launch_bounds__(256) void k_plan_count(PlanArgs a) {
  extern __shared__ int lds[];
  const int n = a.experts + 1;
  const long begin = (long)blockIdx.x * a.at.chunk;
  count_chunk(a, lds, begin, min(begin + a.at.chunk, a.pairs));
  for (int e = threadIdx.x; e < n; e += 256)
    a.plan[a.at.parts + (long)blockIdx.x * n + e] = lds[e] + lds[n + e] + lds[2 * n + e] + lds[3 * n + e];
}

// Each chunk's counts become the counts of the chunks before it; then the offsets and tiles.
__global__ __launch_bounds__(256) void k_plan_sum(PlanArgs a) {
  extern __shared__ int lds[];
  const int n = a.experts + 1;
  for (int e = threadIdx.x; e < n; e += 256) {
    int *parts = a.plan + a.at.parts + e, run = 0;
    for (long c = 0; c < a.at.chunks; c++) {
      const int count = parts[c * n];
      parts[c * n] = run;
      run += count;
    }
    lds[e] = run;
  }
  __syncthreads();
  lay_out(a, lds, lds + n, lds + 2 * n);
}

// The places of a chunk's pairs.  ONE: the only chunk, which does the rest too.
template <bool ONE>
__global__ __launch_bounds__(256) void k_plan_place(PlanArgs a) {
  extern __shared__ int lds[];
  const int n = a.experts + 1, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  int *bins = lds, *counts = lds + WAVES * n, *firsts = counts + n, *work = firsts + n;
  const long begin = (long)blockIdx.x * a.at.chunk, end = min(begin + a.at.chunk, a.pairs);
  count_chunk(a, bins, begin, end);
  if constexpr (ONE) {
    for (int e = threadIdx.x; e < n; e += 256) counts[e] = bins[e] + bins[n + e] + bins[2 * n + e] + bins[3 * n + e];
    __syncthreads();
    lay_out(a, counts, firsts, work);
  }
  // A wave's next place of each expert.
  for (int e = threadIdx.x; e < n; e += 256) {
    int run = ONE ? counts[e] : a.plan[a.at.offsets + e] + a.plan[a.at.parts + (long)blockIdx.x * n + e];
    for (int w = 0; w < WAVES; w++) {
      const int count = bins[w * n + e];
      bins[w * n + e] = run;
      run += count;
    }
  }
  __syncthreads();
  const long part = a.at.chunk / WAVES, from = begin + wave * part, to = min(from + part, end);
  int *next = bins + wave * n;
  for (long p0 = from; p0 < to; p0 += 64) {
    const long p = p0 + lane;
    const bool some = p < to;
    const int e = some ? expert_of(a, p) : -1;
    unsigned long long same = __ballot(some);
    for (int bit = 0; bit < 11; bit++) {
      const unsigned long long set = __ballot(e >> bit & 1);
      same &= e >> bit & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), first = some ? next[e] : 0;
    __builtin_amdgcn_wave_barrier();
    if (some && rank == 0) next[e] = first + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (!some) continue;
    const int at = first + rank;
    a.plan[a.at.order + at] = (int)p;
    a.plan[a.at.place + p] = e < a.experts ? at : -1;
    if (e == a.experts) continue;
    // A tile begins at every TILE_ROWS-th pair of an expert.
    const int begins = ONE ? counts[e] : a.plan[a.at.offsets + e], ends = ONE ? counts[e + 1] : a.plan[a.at.offsets + e + 1];
    for (int s = 0; s < TILE_SIZES; s++) {
      if ((at - begins) % TILE_ROWS[s] != 0) continue;
      const int tile = a.plan[a.at.firsts + (long)s * a.experts + e] + (at - begins) / TILE_ROWS[s];
      *(int4v *)(a.plan + a.at.tiles[s] + 4l * tile) = int4v{e, at, min(at + TILE_ROWS[s], ends), 0};
    }
  }
}

ien_status plan(ien_ctx *ctx, const ien_routes *r) {
  PlanArgs a{r->d_index, r->d_plan, (long)(r->tokens * r->top), (int)r->experts,
             plan_layout(r->tokens, r->experts, r->top)};
  const int n = a.experts + 1;
  const size_t lds = (size_t)((WAVES + 2) * n + WAVES) * 4;
  const dim3 grid((unsigned)a.at.chunks);
  if (a.at.chunks == 1) {
    hipLaunchKernelGGL(k_plan_place<true>, grid, dim3(256), lds, ctx->stream, a);
  } else {
    hipLaunchKernelGGL(k_plan_count, grid, dim3(256), lds, ctx->stream, a);
    hipLaunchKernelGGL(k_plan_sum, dim3(1), dim3(256), lds, ctx->stream, a);
    hipLaunchKernelGGL(k_plan_place<false>, grid, dim3(256), lds, ctx->stream, a);
  }
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

template <typename X>
void route(ien_ctx *ctx, const RouteArgs &a) {
  auto go = [&](auto kernel, int lanes) {
    const int tokens = 256 / lanes;
    const size_t lds = a.kept < a.groups ? (size_t)tokens * (a.experts + a.groups) * sizeof(double) : 0;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.tokens + tokens - 1) / tokens)), dim3(256), lds, ctx->stream, a);
  };
  if (a.experts <= 16) go(k_route<X, 16, 1>, 16);
  else if (a.experts <= 64) go(k_route<X, 16, 4>, 16);
  else if (a.experts <= 128) go(k_route<X, 16, 8>, 16);
  else if (a.experts <= 256) go(k_route<X, 16, 16>, 16);
  else go(k_route<X, 64, 16>, 64);
}

}  // namespace
}  // namespace ien

using namespace ien;

extern "C" {

size_t ien_routes_order(size_t experts) { return 4 * ((experts + 4) / 4); }

size_t ien_routes_ints(size_t tokens, size_t experts, size_t top) {
  if (experts < 1 || experts > MAX_EXPERTS || top < 1 || top > MAX_TOP || tokens > MAX_PAIRS / top) return 0;
  return (size_t)plan_layout(tokens, experts, top).ints;
}

ien_status ien_routes_plan(ien_ctx *ctx, const ien_routes *routes) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  const ien_status s = check_routes(routes, "routes_plan");
  if (s != IEN_OK || routes->tokens == 0) return s;
  return plan(ctx, routes);
}

ien_status ien_route(ien_ctx *ctx, const void *d_logits, ien_out_type type, size_t stride, const ien_router *how,
                     const ien_routes *routes) {
  IEN_CHECK(ctx && how, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(type == IEN_OUT_F16 || type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)type);
  const ien_status s = check_routes(routes, "route");
  if (s != IEN_OK) return s;
  IEN_CHECK(how->score == IEN_SCORE_SOFTMAX || how->score == IEN_SCORE_SIGMOID, IEN_ERR_INPUT, "score %d",
            (int)how->score);
  IEN_CHECK(how->groups >= 1 && routes->experts % how->groups == 0 && how->kept >= 1 && how->kept <= how->groups &&
                (how->group_top == 1 || how->group_top == 2),
            IEN_ERR_INPUT, "%zu experts in %zu groups, %zu kept by their %zu best", routes->experts, how->groups,
            how->kept, how->group_top);
  if (routes->tokens == 0) return IEN_OK;
  IEN_CHECK(d_logits && stride >= routes->experts, IEN_ERR_INPUT, "no logits, or %zu apart for %zu experts", stride,
            routes->experts);
  RouteArgs a{d_logits, (long)stride, (long)routes->tokens, (int)routes->experts, (int)routes->top, how->d_bias,
              how->score == IEN_SCORE_SOFTMAX, (int)how->groups, (int)how->kept, (int)how->group_top,
              how->renormalise, how->scale, routes->d_index, routes->d_weight};
  if (type == IEN_OUT_F16)
    route<_Float16>(ctx, a);
  else
    route<float>(ctx, a);
  IEN_HIP(hipGetLastError());
  return plan(ctx, routes);
}

}  // extern "C"
