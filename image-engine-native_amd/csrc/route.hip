// route.hip -- each token's experts from a router's logits, and the pairs of
// tokens and experts in the order of the experts (ien_route, ien_routes_plan).
//
// Choosing.  16 lanes hold a token's scores (64 where there are more than 256
// experts).  What is not below the (top + 1)-th of the lanes' largest choices, 16
// at most as a rule, is handed a lane each and ordered by counting; else the
// largest choice is found top times.  Equal ones: the lowest index.  Vector
// instructions bound it (over 90 % of the cycles): 65536 tokens, 8 of 256 experts in
// 4 of 8 groups, take 38 us.  Without a bias choices are in the
// order of the logits, which are compared themselves.  With one they are f32
// sums that are off by some steps: where two that matter (neighbours among the
// chosen, the last chosen and the next, the last group kept and the first not)
// are nearer than that, the token is chosen again in f64, by a whole wave: rare but for
// choices that are equal to the last bit (a router of zeros under a bias: 65536 tokens of
// 256 experts 171 us in place of 45, of 8 groups 279 in place of 50).
//
// More than 256 experts go by 64 lanes a token and top + 1 rounds of a maximum over
// them: 65536 tokens, 8 of 300, 512 and 1024 experts 225, 232 and 240 us, of 1024 in
// 32 groups 407.
//
// Planning is a counting sort that keeps the order of equal experts and adds
// nothing atomically across workgroups, so it is the same every time.  The
// workgroups that choose count their chunk's pairs by expert; those that place a
// chunk's pairs add the counts of all chunks (at most 256, from the caches)
// themselves and then take the pairs 64 at a time a wave, a pair's rank among them
// being the number of lanes before it with its expert.  Two launches; up to 64
// tokens take one.

#include <algorithm>
#include <type_traits>

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

// ---- the plan ------------------------------------------------------------------

struct PlanArgs {
  const int *index;
  int *plan;
  long tokens;
  int experts, top;
  PlanLayout at;
};

constexpr int PLACE_WAVES = 8, PLACE_LANES = 64 * PLACE_WAVES;

// What placing a chunk's pairs keeps in LDS, for n = experts + 1 bins: counts of
// each wave's pairs, of the chunks before, of all; the offsets; the first tiles of
// each size; a scan's sums.
struct PlaceShared {
  int *bins, *before, *total, *offsets, *firsts, *sums;
  __device__ PlaceShared(int *p, int n)
      : bins(p), before(bins + PLACE_WAVES * n), total(before + n), offsets(total + n), firsts(offsets + n),
        sums(firsts + TILE_SIZES * n) {}
};
constexpr size_t place_ints(size_t n) {
  return std::max((PLACE_WAVES + 3 + TILE_SIZES) * n + PLACE_WAVES * (TILE_SIZES + 1), (size_t)512);
}

__device__ __forceinline__ int bin_of(int expert, int experts) {
  return (unsigned)expert < (unsigned)experts ? expert : experts;
}

// The sum of v over lanes 0 .. this one: within rows of 16 lanes, then the last lane
// of rows 0 and 2 (row_bcast 15) to 1 and 3, of row 1 (31) to 2 and 3.
__device__ __forceinline__ int sums_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// The offsets and each size's first tiles from the total counts, by the first
// PLACE_LANES threads; into the plan too where `write`.
__device__ void lay_out(const PlanArgs &a, const PlaceShared &s, bool write) {
  constexpr int EACH = ((int)MAX_EXPERTS + 1 + PLACE_LANES - 1) / PLACE_LANES, SUMS = TILE_SIZES + 1;
  const int n = a.experts + 1, tid = threadIdx.x, lane = tid & 63;
  int count[EACH], run[SUMS] = {}, own[SUMS];
  if (tid < PLACE_LANES) {
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int e = tid * EACH + i;
      count[i] = e < n ? s.total[e] : 0;
      run[0] += count[i];
#pragma unroll
      for (int k = 0; k < TILE_SIZES; k++)
        if (e < a.experts) run[k + 1] += (count[i] + TILE_ROWS[k] - 1) / TILE_ROWS[k];
    }
#pragma unroll
    for (int k = 0; k < SUMS; k++) {
      own[k] = run[k];
      run[k] = sums_upto(run[k]);
      if (lane == 63) s.sums[tid / 64 * SUMS + k] = run[k];
    }
  }
  __syncthreads();
  if (tid < PLACE_LANES) {
#pragma unroll
    for (int k = 0; k < SUMS; k++) {
      run[k] -= own[k];
      int all = 0;
#pragma unroll
      for (int w = 0; w < PLACE_WAVES; w++) {
        const int sum = s.sums[w * SUMS + k];
        if (w < tid / 64) run[k] += sum;
        all += sum;
      }
      if (write && k > 0 && tid == 0) a.plan[a.at.totals + k - 1] = all;
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int e = tid * EACH + i;
      if (e >= n) break;
      s.offsets[e] = run[0];
      if (write) a.plan[a.at.offsets + e] = run[0];
      run[0] += count[i];
#pragma unroll
      for (int k = 0; k < TILE_SIZES; k++) {
        s.firsts[k * n + e] = run[k + 1];
        run[k + 1] += (count[i] + TILE_ROWS[k] - 1) / TILE_ROWS[k];
      }
    }
  }
  __syncthreads();
}

// The places of a chunk's pairs, by the first PLACE_WAVES waves, each a part of them
// (expert(p): pair p's of the chunk).  ONE: the only chunk.
template <bool ONE, typename F>
__device__ void place_pairs(const PlanArgs &a, const PlaceShared &s, F expert) {
  const int n = a.experts + 1, tid = threadIdx.x, wave = tid / 64, lane = tid & 63;
  const long begin = (long)blockIdx.x * a.at.chunk * a.top;
  const int pairs = (int)(min((blockIdx.x + 1) * a.at.chunk, a.tokens) * a.top - begin);
  const int part = (pairs + 64 * PLACE_WAVES - 1) / (64 * PLACE_WAVES) * 64;
  const int from = min(wave * part, pairs), to = wave < PLACE_WAVES ? min(from + part, pairs) : from;
  constexpr int HELD = 4;  // a lane's first pairs' experts stay in registers: their loads are under way beside the counts'
  int held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; k++) held[k] = from + 64 * k + lane < to ? expert(from + 64 * k + lane) : 0;
  for (int i = tid; i < (PLACE_WAVES + 2) * n; i += blockDim.x) s.bins[i] = 0;  // (before and total too)
  __syncthreads();
  if constexpr (!ONE) {
    // Four bins a thread, chunks side by side.
    const int fours = (int)a.at.pitch / 4, groups = (int)blockDim.x / fours, four = tid % fours, group = tid / fours;
    int4v before{}, total{};
    if (group < groups) {
#pragma unroll 8
      for (int c = group; c < (int)a.at.chunks; c += groups) {
        const int4v v = *(const int4v *)(a.plan + a.at.parts + (long)c * a.at.pitch + 4 * four);
        total += v;
        if (c < (int)blockIdx.x) before += v;
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * four + i < n) {
          atomicAdd(s.before + 4 * four + i, before[i]);
          atomicAdd(s.total + 4 * four + i, total[i]);
        }
    }
  }
#pragma unroll
  for (int k = 0; k < HELD; k++)
    if (from + 64 * k + lane < to) atomicAdd(s.bins + wave * n + held[k], 1);
  for (int p = from + 64 * HELD + lane; p < to; p += 64) atomicAdd(s.bins + wave * n + expert(p), 1);
  __syncthreads();
  if constexpr (ONE) {
    for (int e = tid; e < n; e += blockDim.x) {
      int sum = 0;
      for (int w = 0; w < PLACE_WAVES; w++) sum += s.bins[w * n + e];
      s.total[e] = sum;
    }
    __syncthreads();
  }
  lay_out(a, s, blockIdx.x == 0);
  // Each wave's next place of each expert.
  for (int e = tid; e < n; e += blockDim.x) {
    int run = s.offsets[e] + s.before[e];
    for (int w = 0; w < PLACE_WAVES; w++) {
      const int count = s.bins[w * n + e];
      s.bins[w * n + e] = run;
      run += count;
    }
  }
  __syncthreads();
  int *next = s.bins + wave * n;
  const int bits = 32 - __clz(a.experts);
  for (int p0 = from; p0 < to; p0 += 64) {
    const int p = p0 + lane;
    const bool some = p < to;
    int e = held[0];
    if (p0 >= from + 64 * HELD) e = some ? expert(p) : 0;
#pragma unroll
    for (int k = 0; k + 1 < HELD; k++) held[k] = held[k + 1];
    unsigned long long same = __ballot(some);
    for (int bit = 0; bit < bits; bit++) {
      const unsigned long long set = __ballot(e >> bit & 1);
      same &= e >> bit & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), first = some ? next[e] : 0;
    __builtin_amdgcn_wave_barrier();
    if (some && rank == 0) next[e] = first + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (!some) continue;
    const int at = first + rank;
    a.plan[a.at.order + at] = (int)(begin + p);
    a.plan[a.at.place + begin + p] = e < a.experts ? at : -1;
    if (e == a.experts) continue;
    // A tile begins at every TILE_ROWS-th pair of an expert.
    const int row = at - s.offsets[e];
#pragma unroll
    for (int k = 0; k < TILE_SIZES; k++)
      if (row % TILE_ROWS[k] == 0)
        *(int4v *)(a.plan + a.at.tiles[k] + 4l * (s.firsts[k * n + e] + row / TILE_ROWS[k])) =
            int4v{e, at, min(at + TILE_ROWS[k], s.offsets[e + 1]), 0};
  }
}

// All of it for up to FEW_PAIRS pairs, a thread a pair: how many come before it is
// counted pair by pair.  expert: their experts in LDS (as many as the next multiple of
// sixteen), begin: room for as many.  (With their choice, of 64 experts: 8 pairs 5.4 us, the general
// way 6.8; 64 pairs 7.6 and 6.9, 128 pairs 10.6 and 6.9.)
constexpr int FEW_PAIRS = 64;
__device__ void place_few(const PlanArgs &a, int *expert, int *begin) {
  const int pairs = (int)a.tokens * a.top, fours = (pairs + 15) / 16 * 4, p = threadIdx.x;
  if (p >= pairs && p < 4 * fours) expert[p] = 1 << 30;  // (none's, after all others)
  __syncthreads();
  const int e = p < pairs ? expert[p] : 0;
  int at = 0, row = 0, all = 0;
  if (p < pairs) {
#pragma unroll 4
    for (int q = 0; q < fours; q++) {
      const int4v v = *(const int4v *)(expert + 4 * q);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        at += v[i] < e;
        all += v[i] == e;
        row += v[i] == e && 4 * q + i < p;
      }
    }
    at += row;
    a.plan[a.at.order + at] = p;
    a.plan[a.at.place + p] = e < a.experts ? at : -1;
  }
  // Whether a tile of each size begins at the pair, a byte each.
  static_assert(TILE_SIZES == 4 && FEW_PAIRS < 256, "counts in bytes");
  unsigned begins = 0;
#pragma unroll
  for (int k = 0; k < TILE_SIZES; k++)
    if (p < pairs && e < a.experts && (row & (TILE_ROWS[k] - 1)) == 0) begins |= 1u << 8 * k;
  if (p < 4 * fours) begin[p] = (int)begins;
  for (int g = threadIdx.x; g <= a.experts; g += blockDim.x) {
    int offset = 0;
#pragma unroll 4
    for (int q = 0; q < fours; q++) {
      const int4v v = *(const int4v *)(expert + 4 * q);
#pragma unroll
      for (int i = 0; i < 4; i++) offset += v[i] < g;
    }
    a.plan[a.at.offsets + g] = offset;
  }
  __syncthreads();
  if (p >= pairs) return;
  unsigned before = 0, total = 0;  // tiles of smaller experts, of all
#pragma unroll 4
  for (int q = 0; q < fours; q++) {
    const int4v v = *(const int4v *)(expert + 4 * q), b = *(const int4v *)(begin + 4 * q);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      total += (unsigned)b[i];
      before += v[i] < e ? (unsigned)b[i] : 0;
    }
  }
#pragma unroll
  for (int k = 0; k < TILE_SIZES; k++) {
    if (p == 0) a.plan[a.at.totals + k] = (int)(total >> 8 * k & 255);
    if (begins >> 8 * k & 1)
      *(int4v *)(a.plan + a.at.tiles[k] + 4l * ((before >> 8 * k & 255) + row / TILE_ROWS[k])) =
          int4v{e, at, min(at + TILE_ROWS[k], at - row + all), 0};
  }
}

__global__ __launch_bounds__(256) void k_plan_count(PlanArgs a) {
  __shared__ int bins[MAX_EXPERTS + 4];
  for (int e = threadIdx.x; e < (int)a.at.pitch; e += 256) bins[e] = 0;
  __syncthreads();
  const long begin = (long)blockIdx.x * a.at.chunk * a.top, end = min((blockIdx.x + 1) * a.at.chunk, a.tokens) * a.top;
  for (long p = begin + threadIdx.x; p < end; p += 256) atomicAdd(bins + bin_of(a.index[p], a.experts), 1);
  __syncthreads();
  for (int e = threadIdx.x; e < (int)a.at.pitch; e += 256) a.plan[a.at.parts + blockIdx.x * a.at.pitch + e] = bins[e];
}

template <bool ONE>
__global__ __launch_bounds__(PLACE_LANES) void k_plan_place(PlanArgs a) {
  extern __shared__ __attribute__((aligned(16))) int lds[];  // (experts are read four at a time)
  const int *index = a.index + (long)blockIdx.x * a.at.chunk * a.top;
  if (ONE && a.tokens * a.top <= FEW_PAIRS) {
    if (threadIdx.x < a.tokens * a.top) lds[threadIdx.x] = bin_of(index[threadIdx.x], a.experts);
    place_few(a, lds, lds + FEW_PAIRS);
    return;
  }
  place_pairs<ONE>(a, PlaceShared(lds, a.experts + 1), [&](int p) { return bin_of(index[p], a.experts); });
}

// ---- choosing ------------------------------------------------------------------

struct RouteArgs {
  const void *logits;
  long stride;
  const float *bias;
  int softmax, groups, kept, group_top, renormalise;
  int by_logit;      // choices are in the order of the logits
  unsigned magic;    // e / (experts a group) = e magic >> 22
  float scale;
  int *index;
  float *weight;
  PlanArgs plan;
};

constexpr float NONE = -__builtin_inff();

// A DPP move of any 4 or 8 bytes.
template <int CTRL, typename T>
__device__ __forceinline__ T moved(T v) {
  if constexpr (sizeof(T) == 8) {
    const long b = __builtin_bit_cast(long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, true);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(T, (unsigned long)hi << 32 | lo);
  } else {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
  }
}
// f(other) for the moves that bring a value over each group of L lanes in halves.
template <int L, typename F>
__device__ __forceinline__ void over_lanes(F f) {
  f([](auto v) { return moved<0xB1>(v); });
  f([](auto v) { return moved<0x4E>(v); });
  f([](auto v) { return moved<0x141>(v); });
  f([](auto v) { return moved<0x140>(v); });
  if constexpr (L == 64) {
    f([](auto v) { return __shfl_xor(v, 16); });
    f([](auto v) { return __shfl_xor(v, 32); });
  }
}
// f(other) for the moves that bring each of 16 lanes the others' values (EVERY: those of each EVERY-th).
template <int EVERY = 1, int N = EVERY, typename F>
__device__ __forceinline__ void round_lanes(F f) {
  f([](auto v) { return moved<0x120 + N>(v); });  // (row_ror)
  if constexpr (N + EVERY < 16) round_lanes<EVERY, N + EVERY>(f);
}
template <int L>
__device__ __forceinline__ int largest(int v) {
  over_lanes<L>([&](auto other) { v = max(v, other(v)); });
  return v;
}
template <int L>
__device__ __forceinline__ int least(int v) {
  over_lanes<L>([&](auto other) { v = min(v, other(v)); });
  return v;
}

// A float as an integer in the same order (both zeros as one), and back: integers are
// compared and moved in one instruction, floats are made quiet first.
__device__ __forceinline__ int key_of_sum(float v) {  // (not of -0, which no sum with a score is)
  const int b = __float_as_int(v);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ int key_of(float v) { return key_of_sum(v + 0.0f); }
__device__ __forceinline__ float value_of(int key) { return __int_as_float(key ^ (key >> 31 & 0x7fffffff)); }
constexpr int NO_KEY = (int)0x807fffff;  // of NONE

// e^x for x <= 88 (0 below -150, e^88 past 88): the hardware's power of two of the rounded x log2(e), times what the
// rounding left (some 2 steps of f32).
__device__ __forceinline__ float exp_f(float x) {
  x = __builtin_amdgcn_fmed3f(x, -150.0f, 88.0f);
  const float hi = x * 1.44269502f, lo = fmaf(x, 1.44269502f, -hi) + x * 1.92596303e-8f;
  const float r = __builtin_amdgcn_exp2f(hi);
  return fmaf(r * lo, 0.693147181f, r);
}
// Of a key and what goes before it where keys are equal, the lower first.
__device__ __forceinline__ long ordered(int key, int at) { return (long)key << 32 | (unsigned)~at; }

// The two largest keys of two lanes.
__device__ __forceinline__ void merge(int &best, int &next, int b, int n) {
  next = max(max(next, n), min(best, b));
  best = max(best, b);
}
// From every lane's two largest keys of G groups the 16 lanes' of one: of group lane G / 16, in best[0] and next[0].
// Lanes share the groups out as they go, half of them each, until one is left (8 groups: 8 merges in place of 32).
template <int G, int BIT = 8>
__device__ __forceinline__ void share_out(int *best, int *next, int lane) {
  constexpr int CTRL = BIT == 8 ? 0x140 : BIT == 4 ? 0x141 : BIT == 2 ? 0x4E : 0xB1;  // (within the lanes that have the same groups)
  const bool upper = lane & BIT;
#pragma unroll
  for (int g = 0; g < (G + 1) / 2; g++) {
    int b = best[g], n = next[g];
    if constexpr (G > 1) {
      b = upper ? best[g] : best[g + G / 2];
      n = upper ? next[g] : next[g + G / 2];
      best[g] = upper ? best[g + G / 2] : best[g];
      next[g] = upper ? next[g + G / 2] : next[g];
    }
    merge(best[g], next[g], moved<CTRL>(b), moved<CTRL>(n));
  }
  if constexpr (BIT > 1) share_out<(G + 1) / 2, BIT / 2>(best, next, lane);
}

__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One token's choice in f64 by a whole wave, V experts a lane: lane k's is slot k's
// expert and weight.  by_logit: the weights of the experts that lanes hold in `chosen`.
template <typename X, int V>
__device__ __forceinline__ void choose_f64(const RouteArgs &a, const X *row, double *ranks, int lane, int &chosen, float &weight) {
  constexpr int L = 64;
  const int experts = a.plan.experts, top = a.plan.top;
  const double none = -__builtin_inf();
  auto logit = [&](int e) {
    const double v = e < experts ? (double)row[e] : none;
    return v > none ? v : none;  // (NaN too)
  };
  double m = none, sum = 0.0;
  if (a.softmax) {
    for (int e = lane; e < experts; e += L) m = fmax(m, logit(e));
    over_lanes<L>([&](auto other) { m = fmax(m, other(m)); });
  }
  auto score = [&](double v) {
    if (v == none) return 0.0;
    if (!a.softmax) return 1.0 / (1.0 + exp(-v));
    return v == m ? 1.0 : exp(v - m);  // (infinite ones share all)
  };
  double c[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    c[i] = score(logit(lane + L * i));
    sum += c[i];
  }
  if (a.softmax) {
    over_lanes<L>([&](auto other) { sum += other(sum); });
  } else {
    sum = 1.0;
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + L * i;
    const float b = a.bias && e < experts ? a.bias[e] : 0.0f;
    c[i] = logit(e) == none || !(b > NONE) ? none : c[i] / sum + (double)b;
  }
  if (a.kept < a.groups) {
    for (int g = 0; g < a.groups; g++) {
      double best = none, next = none;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (((lane + L * i) * a.magic) >> 22 == (unsigned)g) next = fmax(next, fmin(best, c[i])), best = fmax(best, c[i]);
      over_lanes<L>([&](auto other) {
        const double b = other(best), n = other(next);
        next = fmax(fmax(next, n), fmin(best, b));
        best = fmax(best, b);
      });
      if (lane == 0) ranks[g] = a.group_top == 2 && next > none ? best + next : best;
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < V; i++) {
      if (lane + L * i >= experts) continue;
      const int mine = (lane + L * i) * a.magic >> 22;
      const double rank = ranks[mine];
      int ahead = 0;
      for (int g = 0; g < a.groups; g++) ahead += before(ranks[g], g, rank, mine);
      if (ahead >= a.kept) c[i] = none;
    }
    wave_fence();
  }
  if (!a.by_logit) chosen = -1;
  for (int k = 0; k < (a.by_logit ? 0 : top); k++) {
    double best = none;
    int at = 1 << 30;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (c[i] > best) best = c[i], at = lane + L * i;
    over_lanes<L>([&](auto other) {
      const double that = other(best);
      const int there = other(at);
      if (before(that, there, best, at)) best = that, at = there;
    });
#pragma unroll
    for (int i = 0; i < V; i++)
      if (lane + L * i == at) c[i] = none;
    if (lane == k && best > none) chosen = at;
  }
  const double s = chosen >= 0 ? score(logit(chosen)) / sum : 0.0;
  double total = s;
  over_lanes<L>([&](auto other) { total += other(total); });
  const double w = !a.renormalise ? s : total > 0.0 ? s / total : 0.0;
  weight = (float)(w * (double)a.scale);
}

constexpr int route_lanes(int l) { return l == 16 ? 1024 : 512; }  // of a workgroup (64 lanes a token: f64 ranks of all groups fit)

// L lanes a token, V experts a lane: expert l + L i.  A workgroup takes a chunk of
// tokens, so many at a time.  ONE: the only chunk, whose pairs it places too.
template <typename X, int L, int V, bool ONE>
__global__ __launch_bounds__(route_lanes(L)) void k_route(RouteArgs a) {
  constexpr int LANES = route_lanes(L), TOKENS = LANES / L;
  extern __shared__ __attribute__((aligned(16))) int lds[];  // (experts four at a time, ranks in f64; behind the arrays below)
  constexpr int LISTS = L == 16 ? TOKENS * 16 : 1;
  __shared__ int candidates[3 * LISTS];  // the keys of a token's, their scores, their experts
  __shared__ int boards[TOKENS * (L * V + 16)];  // a token's keys (16 more: a wave's four then write to different banks)
  __shared__ int taken_tokens;
  __shared__ float biases[L * V];
  const int experts = a.plan.experts, top = a.plan.top, n = experts + 1;
  int tid = threadIdx.x;
  int *bins = lds;                                      // the chunk's counts; ONE: its pairs' experts
  const int held = ONE ? 64 * top : (int)a.plan.at.pitch;  // (whole fours)
  float *ranks = (float *)(lds + held);                   // [token][groups]; f64 of one token a wave
  if constexpr (!ONE) {
    for (int e = threadIdx.x; e < held; e += LANES) bins[e] = 0;
  }
  for (int e = threadIdx.x; e < L * V; e += LANES) {
    const float b = a.bias && e < experts ? a.bias[e] : 0.0f;
    biases[e] = b > NONE ? b : NONE;  // (NaN too)
  }
  if (threadIdx.x == 0) taken_tokens = 0;
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);  // (else the barrier waits for what every wave computes below: a token 5.8 us, so 5.3)
  const long begin = (long)blockIdx.x * a.plan.at.chunk, end = min(begin + a.plan.at.chunk, a.plan.tokens);
  for (;;) {
    // (What follows from it is cheaper to compute again than to keep: 48 registers too many.)
    if constexpr (V == 16) asm volatile("" : "+v"(tid));
    int lane = tid % L;
    if constexpr (V < 16) asm volatile("" : "+v"(lane));
    const int slot = tid / L;
    // The next of the chunk's tokens that no wave has (a wave may be held up by a choice in f64).
    int next = 0;
    if ((tid & 63) == 0) next = atomicAdd(&taken_tokens, 64 / L);
    const long t0 = begin + __builtin_amdgcn_readfirstlane(next);
    if (t0 >= end) break;
    const long t = min(t0 + slot % (64 / L), end - 1);
    const bool some = t0 + slot % (64 / L) < end;
    const X *row = (const X *)a.logits + t * a.stride;
    float s[V];
    int c[V];  // the choices' keys
    if (experts == L * V) {  // (one address, and what is constant from it)
      row += lane;
#pragma unroll
      for (int i = 0; i < V; i++) s[i] = (float)row[L * i];
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) {
        s[i] = (float)row[min(lane + L * i, experts - 1)];
        s[i] = lane + L * i < experts ? s[i] : NONE;
      }
    }
    unsigned most = 0, gone = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      s[i] = s[i] > NONE ? s[i] : NONE;  // (NaN too)
      most = max(most, __float_as_uint(s[i]));
    }
    if (!a.by_logit && __ballot(most == __float_as_uint(NONE))) {  // (it is the last of them as an integer)
#pragma unroll
      for (int i = 0; i < V; i++) gone |= (s[i] == NONE ? 1u : 0u) << i;
    }
    if (a.softmax || a.by_logit) {
#pragma unroll
      for (int i = 0; i < V; i++) c[i] = key_of(s[i]);
    }
    // How far a score may be off, in halves of a step of 1: of a logistic function 4 of its exponential, at most
    // a quarter of which reaches it, a step of the reciprocal and two roundings; of a softmax 0.4 of the argument
    // (d e^-d of its rounding), and of the largest score 4 of the exponential, as much of the sum's, 7 of their
    // arguments, 21 of the additions and 2 of the quotient.
    float off = 5.0f;
    if (a.softmax) {
      int key = NO_KEY;
#pragma unroll
      for (int i = 0; i < V; i++) key = max(key, c[i]);
      const float m = value_of(largest<L>(key));
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) {
        s[i] = exp_f(s[i] == m ? 0.0f : s[i] - m);  // (infinite ones share all)
        sum += s[i];
      }
      sum = group_sum<L>(sum);
      const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
      off = 0.4f + 38.0f * inv;
#pragma unroll
      for (int i = 0; i < V; i++) s[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) {
        s[i] = __builtin_amdgcn_rcpf(1.0f + exp_f(-s[i]));  // (under 1e-30, also where it is less than that still)
      }
    }
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < V; i++) c[i] = key_of_sum(s[i] + biases[lane + L * i]);
    } else if (!a.by_logit) {
#pragma unroll
      for (int i = 0; i < V; i++) c[i] = __float_as_int(s[i]);  // (none is negative)
    }
    if (__ballot(gone)) {
#pragma unroll
      for (int i = 0; i < V; i++) c[i] = gone >> i & 1 ? NO_KEY : c[i];
    }
    // Two choices that are nearer than this may be in the other order: each is off by its score's error and its own
    // rounding, half a step of its size.  (That bound grows with a choice, so what is clear between neighbours in
    // order is clear between all.  The factor is a step and what the comparison's own roundings come to.)
    auto close = [&](float larger, float smaller) {
      return larger - smaller < 0x1.0001p-23f * (off + fmaxf(fabsf(larger), fabsf(smaller)));
    };
    bool unclear = false;
    if (a.kept < a.groups) {
      const int per = experts / a.groups;
      // Of two choices half their sum, which f32 always holds (two of its lowest values sum to what is no expert's).
      float cancelled = 0.0f;  // the part of two choices that is not in their sum's size
      auto rank_of = [&](int best, int next) {
        if (a.group_top == 1) return best;
        const float b = 0.5f * value_of(best), n = next > NO_KEY ? 0.5f * value_of(next) : 0.0f;
        cancelled = fmaxf(cancelled, fminf(b, -n));
        return key_of(b + n);
      };
      // The least that a kept group's rank may be, the most that another's: it is off by the choices' errors, half a step
      // of their sizes for the choices' roundings and another for the sum's, and the bound's own.  (An infinite
      // one stays infinite.)
      auto bound = [&](bool keep, int rank) {
        const float r = value_of(rank);
        const float by = 0x1.0001p-23f * (0.5f * off + 1.5f * fminf(fabsf(r), 0x1.fffffep127f) + 3.0f * cancelled);
        return key_of(keep ? r - by : r + by);
      };
      int low = 0x7fffffff, high = NO_KEY;  // of the groups kept, and of the others
      // A group is OF of every lane's experts, one after another: G groups, the last of them of no expert perhaps.
      auto in_lanes = [&](auto of) {
        constexpr int OF = decltype(of)::value, G = V / OF, EVERY = 16 / G;
        int best[G], next[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
          best[g] = c[g * OF], next[g] = NO_KEY;
#pragma unroll
          for (int i = 1; i < OF; i++) {
            next[g] = max(next[g], min(best[g], c[g * OF + i]));
            best[g] = max(best[g], c[g * OF + i]);
          }
        }
        share_out<G>(best, next, lane);
        if constexpr (L == 64) {
          merge(best[0], next[0], __shfl_xor(best[0], 16), __shfl_xor(next[0], 16));
          merge(best[0], next[0], __shfl_xor(best[0], 32), __shfl_xor(next[0], 32));
        }
        const int group = lane % 16 / EVERY, own = rank_of(best[0], next[0]);
        const long mine = ordered(own, group);
        int ahead = 0;
        round_lanes<EVERY>([&](auto other) { ahead += other(mine) > mine; });
        const bool keep = ahead < a.kept && group < a.groups;
        if (group < a.groups) (keep ? low : high) = bound(keep, own);
        const unsigned kept = (unsigned)(__ballot(keep) >> (L == 16 ? slot % 4 * 16 : 0));
#pragma unroll
        for (int i = 0; i < V; i++) {
          const int mask = (int)(kept << (31 - i / OF * EVERY)) >> 31;
          c[i] = (c[i] & mask) | (NO_KEY & ~mask);
        }
      };
      if (V >= 2 && per == L) {
        if constexpr (V >= 2) in_lanes(std::integral_constant<int, 1>{});
      } else if (V >= 4 && per == 2 * L) {
        if constexpr (V >= 4) in_lanes(std::integral_constant<int, 2>{});
      } else if (V >= 8 && per == 4 * L) {
        if constexpr (V >= 8) in_lanes(std::integral_constant<int, 4>{});
      } else if (V >= 16 && per == 8 * L) {
        if constexpr (V >= 16) in_lanes(std::integral_constant<int, 8>{});
      } else {
        // Through LDS: a group's experts are read by `share` lanes beside each other (65536 tokens, with their plan: 32
        // groups of 8 experts 88 us, 10 of 20 66; every group looked for among all lanes' experts 157 and 82).
        int *mine = (int *)ranks + (L == 16 ? 1 : 2) * slot * a.groups, *board = boards + slot * (L * V + 16);
#pragma unroll
        for (int i = 0; i < V; i++) board[lane + L * i] = c[i];
        wave_fence();
        const int share_bits = max(0, (L == 16 ? 4 : 6) - (32 - __clz(a.groups - 1))), share = 1 << share_bits;
        const int part = lane & (share - 1), group = lane >> share_bits;
        auto rank_in = [&](int g) {
          int best = NO_KEY, next = NO_KEY;
          for (int e = g < a.groups ? part : per; e < per; e += share) {
            const int v = board[g * per + e];
            next = max(next, min(best, v));
            best = max(best, v);
          }
          int steps = share_bits;
          over_lanes<L>([&](auto other) {
            if (steps-- > 0) merge(best, next, other(best), other(next));
          });
          return rank_of(best, next);
        };
        if (a.groups <= L) {
          const int own = rank_in(group);
          const bool its = part == 0 && group < a.groups;
          int ahead = 0;
          if constexpr (L == 16) {
            const long rank = its ? ordered(own, group) : (long)(1ull << 63);
            round_lanes([&](auto other) { ahead += other(rank) > rank; });
          } else {
            for (int g = 0; g < a.groups; g++) {
              const int rank = __shfl(own, g << share_bits);
              ahead += rank > own || (rank == own && g < group);
            }
          }
          if (its) {
            (ahead < a.kept ? low : high) = bound(ahead < a.kept, own);
            mine[group] = ahead < a.kept;
          }
        } else {
          for (int g = lane; g < a.groups; g += L) mine[g] = rank_in(g);
          wave_fence();
          unsigned long long keep = 0;  // of this lane's groups lane + L j
          for (int j = 0; lane + L * j < a.groups; j++) {
            const int rank = mine[lane + L * j];
            int ahead = 0;
            for (int g = 0; g < a.groups; g++) ahead += mine[g] > rank || (mine[g] == rank && g < lane + L * j);
            if (ahead < a.kept)
              keep |= 1ull << j, low = min(low, bound(true, rank));
            else
              high = max(high, bound(false, rank));
          }
          wave_fence();
          for (int j = 0; lane + L * j < a.groups; j++) mine[lane + L * j] = (int)(keep >> j & 1);
        }
        wave_fence();
#pragma unroll
        for (int i = 0; i < V; i++)
          if (lane + L * i < experts && mine[(lane + L * i) * a.magic >> 22] == 0) c[i] = NO_KEY;
        wave_fence();
      }
      low = least<L>(low), high = largest<L>(high);
      unclear = high > NO_KEY && low < high;
    }
    // A lane's expert and score, and which slot they are for: the slots' are the first `top`.
    int chosen = -1, place = lane;
    bool any = false, choose = true;
    float score = 0.0f, total = 0.0f;
    if constexpr (L == 16) {
      // By counting.  At least top + 1 choices are as large as the (top + 1)-th of the lanes' largest; where they
      // are 16 at most, as they mostly are, every lane takes one and counts those before it.
      int mine = NO_KEY;
#pragma unroll
      for (int i = 0; i < V; i++) mine = max(mine, c[i]);
      int ahead = 0;
      round_lanes([&](auto other) { ahead += other(mine) > mine; });
      const int from = max(least<L>(ahead <= top ? mine : 0x7fffffff), NO_KEY + 1);
      int upto = 0, own;
#pragma unroll
      for (int i = 0; i < V; i++) upto += c[i] >= from;
      own = upto;
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xF, 0xF, true);  // (row_shr 1, 2, 4, 8: sums from lane 0 on)
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xF, 0xF, true);
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xF, 0xF, true);
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xF, 0xF, true);
      if (top < 16 && !__ballot(upto > 16)) {
        int *const first = candidates + slot * 16, *at = first + upto - own;
        first[lane] = NO_KEY;
        first[lane + 2 * LISTS] = (int)MAX_EXPERTS + lane;
        wave_fence();
#pragma unroll
        for (int i = 0; i < V; i++)
          if (c[i] >= from) {
            at[0] = c[i], at[LISTS] = __float_as_int(s[i]), at[2 * LISTS] = lane + L * i;
            at++;
          }
        wave_fence();
        const int key = first[lane], expert = first[lane + 2 * LISTS];
        const float its = __int_as_float(first[lane + LISTS]);  // (past the candidates: not used)
        const long mine = ordered(key, expert);
        place = 0;
        round_lanes([&](auto other) { place += other(mine) > mine; });
        const bool taken = place < top && key > NO_KEY;
        if (taken) chosen = expert, score = its;
        if (!a.by_logit) {  // (in their order each is compared with the next one)
          wave_fence();
          first[place] = key;
          wave_fence();
          const int near = taken && close(value_of(key), value_of(first[place + 1]));
          unclear = unclear || largest<L>(near);
        }
        total = group_sum<L>(score);
        any = largest<L>(key) > NO_KEY;
        choose = false;
      }
    }
    if (choose) {  // slot k's stay with lane k
      float last = __builtin_inff();
      for (int k = 0; k <= top; k++) {
        int key = NO_KEY;
#pragma unroll
        for (int i = 0; i < V; i++) key = max(key, c[i]);
        key = largest<L>(key);
        const float best = value_of(key);
        if (key > NO_KEY && close(last, best)) unclear = true;
        last = best;
        any = any || key > NO_KEY;
        if (k == top) break;
        int at = 1 << 30;
        float its = 0.0f;
#pragma unroll
        for (int i = V - 1; i >= 0; i--)
          if (c[i] == key) at = lane + L * i, its = s[i];
        const int first = least<L>(at);
        const bool owner = first == at;
#pragma unroll
        for (int i = 0; i < V; i++)
          if (first == lane + L * i) c[i] = NO_KEY;
        its = group_sum<L>(owner && key > NO_KEY ? its : 0.0f);
        total += its;
        if (lane == k && key > NO_KEY) chosen = first, score = its;
      }
    }
    float weight = (!a.renormalise ? score : total > 0.0f ? score / total : 0.0f) * a.scale;
    // (f32 scores that vanish: their shares need not.)
    unclear = (unclear && !a.by_logit) || (a.renormalise && total < 1e-30f && any);
    for (unsigned long long left = __ballot(unclear); left != 0;) {
      const int first = __ffsll(left) - 1, token = first / L;  // (the wave's)
      left &= ~((L == 64 ? ~0ull : (1ull << (L & 63)) - 1) << token * L);
      const long there = __shfl(t, first);
      const bool mine = slot % (64 / L) == token;
      int c64 = mine ? chosen : -1;
      float w64;
      choose_f64<X, (L * V + 63) / 64>(a, (const X *)a.logits + there * a.stride,
                                       (double *)(ranks + (L == 16 ? slot / 4 * 4 : 2 * slot) * a.groups), tid & 63, c64, w64);
      if (!a.by_logit) {
        c64 = __shfl(c64, lane);
        w64 = __shfl(w64, lane);
        if (mine) chosen = c64, place = lane;
      }
      if (mine) weight = w64;
    }
    if (some && place < top) {
      const long pair = t * top + place;
      a.index[pair] = chosen;
      a.weight[pair] = weight;
      if constexpr (ONE)
        bins[pair] = bin_of(chosen, experts);
      else
        atomicAdd(bins + bin_of(chosen, experts), 1);
    }
    wave_fence();  // (the ranks' next token)
  }
  __syncthreads();
  if (ONE && a.plan.tokens * top <= FEW_PAIRS)
    place_few(a.plan, bins, lds + held);
  else if constexpr (ONE)
    place_pairs<true>(a.plan, PlaceShared(lds + held, n), [&](int p) { return bins[p]; });
  else
    for (int e = threadIdx.x; e < held; e += LANES) a.plan.plan[a.plan.at.parts + blockIdx.x * a.plan.at.pitch + e] = bins[e];
}

void launch_place(ien_ctx *ctx, const PlanArgs &a) {
  const size_t lds = place_ints((size_t)a.experts + 1) * 4;
  if (a.at.chunks == 1)
    hipLaunchKernelGGL(k_plan_place<true>, dim3(1), dim3(PLACE_LANES), lds, ctx->stream, a);
  else
    hipLaunchKernelGGL(k_plan_place<false>, dim3((unsigned)a.at.chunks), dim3(PLACE_LANES), lds, ctx->stream, a);
}

template <typename X, int L, int V>
void launch_route(ien_ctx *ctx, const RouteArgs &a) {
  const PlanArgs &p = a.plan;
  const bool one = p.at.chunks == 1;
  const size_t held = one ? 64 * (size_t)p.top : (size_t)p.at.pitch;
  size_t ints = a.kept < a.groups ? (size_t)(route_lanes(L) / L) * a.groups * (L == 16 ? 1 : 2) : 0;
  if (one) ints = std::max(ints, place_ints((size_t)p.experts + 1));
  const size_t lds = (held + ints) * 4;
  if (one)
    hipLaunchKernelGGL((k_route<X, L, V, true>), dim3(1), dim3(route_lanes(L)), lds, ctx->stream, a);
  else
    hipLaunchKernelGGL((k_route<X, L, V, false>), dim3((unsigned)p.at.chunks), dim3(route_lanes(L)), lds, ctx->stream, a);
}

template <typename X>
void route(ien_ctx *ctx, const RouteArgs &a) {
  const int experts = a.plan.experts;
  if (experts <= 16) launch_route<X, 16, 1>(ctx, a);
  else if (experts <= 64) launch_route<X, 16, 4>(ctx, a);
  else if (experts <= 128) launch_route<X, 16, 8>(ctx, a);
  else if (experts <= 256) launch_route<X, 16, 16>(ctx, a);
  else launch_route<X, 64, 16>(ctx, a);
}

PlanArgs plan_args(const ien_routes *r) {
  return {r->d_index, r->d_plan, (long)r->tokens, (int)r->experts, (int)r->top,
          plan_layout(r->tokens, r->experts, r->top)};
}

}  // namespace
}  // namespace ien

using namespace ien;

extern "C" {

size_t ien_routes_order(size_t experts) { return 4 * ((experts + 4) / 4); }

size_t ien_routes_ints(size_t tokens, size_t experts, size_t top) {
  if (experts < 1 || experts > MAX_EXPERTS || top < 1 || top > MAX_TOP || top > experts || tokens > MAX_PAIRS / top) return 0;
  return (size_t)plan_layout(tokens, experts, top).ints;
}

ien_status ien_routes_plan(ien_ctx *ctx, const ien_routes *routes) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  const ien_status s = check_routes(routes, "routes_plan");
  if (s != IEN_OK || routes->tokens == 0) return s;
  const PlanArgs a = plan_args(routes);
  if (a.at.chunks > 1) {
    hipLaunchKernelGGL(k_plan_count, dim3((unsigned)a.at.chunks), dim3(256), 0, ctx->stream, a);
    IEN_HIP(hipGetLastError());
  }
  launch_place(ctx, a);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
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
  const unsigned per = (unsigned)(routes->experts / how->groups);
  const bool grouped = how->kept < how->groups;
  // (e magic is e / per + e (magic - 2^22 / per) / 2^22, and e per < 2^22: the second part is under 1 / per.)
  RouteArgs a{d_logits, (long)stride, how->d_bias, how->score == IEN_SCORE_SOFTMAX, (int)how->groups, (int)how->kept,
              (int)how->group_top, how->renormalise, !how->d_bias && !(grouped && how->group_top == 2),
              ((1u << 22) + per - 1) / per, how->scale, routes->d_index, routes->d_weight, plan_args(routes)};
  if (type == IEN_OUT_F16)
    route<_Float16>(ctx, a);
  else
    route<float>(ctx, a);
  IEN_HIP(hipGetLastError());
  if (a.plan.at.chunks > 1) launch_place(ctx, a.plan);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

}  // extern "C"
