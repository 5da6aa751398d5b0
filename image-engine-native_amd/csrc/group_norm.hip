// group_norm.hip -- group norm with an activation over channels-last maps
// (ien_group_norm, ien_group_norm8): y = act((x - m) / sqrt(v + eps) gamma +
// beta) with m and v over a map's pixels and a group's channels.
//
// A lane keeps eight consecutive channels of every px-th pixel, so a pixel is
// read in 16-byte pieces whatever the groups, and holds a mean and the squares
// of the deviations from it for each of its channels.  A batch of pixels in
// registers gives both exactly as defined (first the mean, then the squares);
// batches, lanes and workgroups join by
//   m = m1 + d n2 / n,  q = q1 + q2 + d^2 n1 n2 / n,  d = m2 - m1, n = n1 + n2
// (Chan, Golub and LeVeque), which cancels nothing, wherever the mean lies, and
// channels of a group by the same with equal counts.  The order is fixed by the
// sizes alone.
//
// Memory bounds it: x is read for the statistics, read again and y written.  The
// two passes share a split of the pixels, and the second takes each part from
// its end, so that some of it is still in the L2 of its XCD; the rest comes from
// the memory-side cache where x fits that.  512 x 768 x 128 in f16: 21 + 37 us,
// 5.3 TB/s of the three passes.  Maps of a few hundred pixels take one launch, a
// workgroup a few groups (16 x 16 x 512: 7.2 us).  Lanes to spare are what narrow
// rows cost, most into 8 bits, where a pixel takes 16 (50000 x 8: 14.7 us into f16,
// 55.5 into 8 bits).

#include <algorithm>

#include "eight_bits.h"

namespace ien {
namespace {

struct NormArgs {
  const void *x;
  long pixels, stride;
  int c, groups, act;
  const float *gamma, *beta;
  float eps;
  void *y;
  long ystride;
  uint8_t *scales;
  long scale_stride;
  int span;     // channels a workgroup handles (c, or a part in one launch)
  int px;       // pixels side by side in one launch
  int chunks;   // parts of an image's pixels
  long chunk;   // pixels of a part
  float2 *part;  // [image][chunk][group]: mean and squares
};

constexpr int LANES = 1024;  // of a workgroup, at most

// LDS of a workgroup's lanes while they join: a count, and the means and
// squares of up to eight runs of channels, [run][lane].
struct Shared {
  float *n, *m, *q;
  int lanes;
  __device__ __forceinline__ Shared(float *p) : n(p), m(p + blockDim.x), q(m + 8 * blockDim.x), lanes(blockDim.x) {}
};
inline size_t shared_floats(int lanes) { return (size_t)17 * lanes; }

// (m1, q1) of n1 joined with (m2, q2): w = n2 / (n1 + n2), nw = n1 w.
__device__ __forceinline__ void join(float &m1, float &q1, float m2, float q2, float w, float nw) {
  const float d = m2 - m1;
  m1 += d * w;
  q1 += q2 + d * d * nw;
}
// n2 / n (1 ulp: where both means agree it does not matter).
__device__ __forceinline__ float share(float n2, float n) { return n > 0.0f ? n2 * __builtin_amdgcn_rcpf(n) : 0.0f; }

// `eights` lanes a pixel, px pixels side by side.
struct Place {
  int eights, px, slot, eight;
  __device__ __forceinline__ Place(int span, int round, int pixels) {
    eights = (span / 8 + (span % 8 != 0) + round - 1) / round * round;
    px = pixels ? pixels : (int)blockDim.x / eights;
    slot = threadIdx.x / eights;
    eight = threadIdx.x - slot * eights;
    if (slot >= px) eight = eights;  // (idle)
  }
};

// Eight channels of a pixel as they are; past the end the last one again (no
// result is made of those).  EIGHTS: c is in eights, and no branch stands between
// the loads of a batch.  Otherwise none does either in narrow rows, whose
// values are read one by one: a branch would wait for the loads before it.
template <typename T>
using Eight = T __attribute__((ext_vector_type(8)));
template <bool EIGHTS, typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *row, int at, int c) {
  typedef Eight<T> Any __attribute__((aligned(sizeof(T))));
  if (EIGHTS) return *(const Any *)(row + min(at, c - 8));
  if (c >= 64 && at + 8 <= c) return *(const Any *)(row + at);
  Eight<T> v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = row[min(at + i, c - 1)];
  return v;
}

// U pixels' values, the first `many` of them counted (ALL: all), into a lane's
// statistics.
template <bool ALL, int U>
__device__ __forceinline__ void take(const float (&v)[U][8], int many, float &n, float (&m)[8], float (&q)[8]) {
  // (The first batch is taken as it is: k rcp(k) may be a step off 1.)
  const float k = ALL ? (float)U : (float)many, w = n > 0.0f ? share(k, n + k) : 1.0f, nw = n * w;
  float counts[U];
#pragma unroll
  for (int u = 0; u < U; u++) counts[u] = u < many ? 1.0f : 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // (Sums from the first value on: of equal ones exact.)
    float s = 0.0f, e = 0.0f;
#pragma unroll
    for (int u = 1; u < U; u++) s += ALL ? v[u][i] - v[0][i] : (v[u][i] - v[0][i]) * counts[u];
    const float mean = v[0][i] + (ALL ? s * (1.0f / U) : s * __builtin_amdgcn_rcpf(k));
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float d = v[u][i] - mean;
      e += ALL ? d * d : d * d * counts[u];
    }
    join(m[i], q[i], mean, e, w, nw);
  }
  n += k;
}

// The lanes' statistics of the workgroup's channels, joined by group: f(group
// of the span, mean, squares), one lane a group.  Channels first, where a lane's
// eight have a group in common: runs of W = gcd(per, 8) channels.
template <typename F>
__device__ __forceinline__ void by_group(const Shared &s, const Place &p, float n, float (&m)[8], float (&q)[8], int span,
                                         int per, F f) {
  const int t = threadIdx.x, W = per & 7 ? per & -per : 8, runs = 8 / W;
  auto pairs = [&](auto width) {  // runs of `width` to runs of twice as many
    constexpr int V = decltype(width)::value;
#pragma unroll
    for (int i = 0; i < 4 / V; i++) {
      const float a = m[2 * i], b = m[2 * i + 1], d = b - a;
      m[i] = a + 0.5f * d;
      q[i] = q[2 * i] + q[2 * i + 1] + d * d * (0.5f * V * n);
    }
  };
  if (W >= 2) pairs(Act<1>{});
  if (W >= 4) pairs(Act<2>{});
  if (W >= 8) pairs(Act<4>{});
  s.n[t] = n;
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < runs) s.m[i * s.lanes + t] = m[i], s.q[i * s.lanes + t] = q[i];
  int width = 1;
  while (width < p.px) width *= 2;
  for (int w = width / 2; w >= 1; w /= 2) {
    __syncthreads();
    if (p.slot < w && p.slot + w < p.px) {
      const int o = t + w * p.eights;
      const float n2 = s.n[o], k = share(n2, n + n2), nk = W * n * k;
      n += n2;
      s.n[t] = n;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < runs) {
          join(m[i], q[i], s.m[i * s.lanes + o], s.q[i * s.lanes + o], k, nk);
          s.m[i * s.lanes + t] = m[i], s.q[i * s.lanes + t] = q[i];
        }
    }
  }
  __syncthreads();
  const float each = s.n[0] * W;  // values of a run
  const int many = per / W;       // runs of a group
  auto at = [&](int r) { return (r & (runs - 1)) * s.lanes + r / runs; };
  if (many <= 8) {
    for (int g = t; g < span / per; g += s.lanes) {
      const float base = s.m[at(g * many)];  // (sums from it on: of equal means exact)
      float mean = 0.0f, squares = 0.0f;
      for (int r = 1; r < many; r++) mean += s.m[at(g * many + r)] - base;
      mean = base + mean / (float)many;
      for (int r = 0; r < many; r++) {
        const float d = s.m[at(g * many + r)] - mean;
        squares += s.q[at(g * many + r)] + each * d * d;
      }
      f(g, mean, squares);
    }
  } else {
    for (int g = t >> 6; g < span / per; g += s.lanes >> 6) {
      const float base = s.m[at(g * many)];
      float mean = 0.0f, squares = 0.0f;
      for (int r = t & 63; r < many; r += 64) mean += s.m[at(g * many + r)] - base;
      mean = base + group_sum<64>(mean) / (float)many;
      for (int r = t & 63; r < many; r += 64) {
        const float d = s.m[at(g * many + r)] - mean;
        squares += s.q[at(g * many + r)] + each * d * d;
      }
      squares = group_sum<64>(squares);
      if ((t & 63) == 0) f(g, mean, squares);
    }
  }
}

// A lane's statistics of its `left` pixels from x on, `step` apart.
template <bool EIGHTS, typename T>
__device__ __forceinline__ void gather(const T *x, long step, int left, int at, int c, float &n, float (&m)[8],
                                       float (&q)[8]) {
  constexpr int U = (sizeof(T) == 2 ? 8 : 4) / (EIGHTS ? 1 : 2);  // (single values take a register each)
  auto batch = [&](auto all) {
    constexpr bool ALL = decltype(all)::value;
    Eight<T> x8[U];
#pragma unroll
    for (int u = 0; u < U; u++) x8[u] = load_eight<EIGHTS>(x + (ALL || u < left ? u : 0) * step, at, c);
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[u][i] = (float)x8[u][i];
    take<ALL>(v, left, n, m, q);
  };
  for (; left >= U; left -= U, x += U * step) batch(Act<1>{});
  if (left > 0) batch(Act<0>{});
}

// A part of an image's pixels: its groups' means and squares.
template <typename T, bool EIGHTS>
__global__ __launch_bounds__(LANES) void k_norm_stats(NormArgs a) {
  extern __shared__ float lds[];
  const Shared s(lds);
  const Place p(a.c, 1, 0);
  const int image = blockIdx.x / a.chunks, part = blockIdx.x % a.chunks, at = p.eight * 8;
  const long begin = part * a.chunk;
  const int many = (int)min(a.chunk, a.pixels - begin);
  const T *x = (const T *)a.x + (image * a.pixels + begin + p.slot) * a.stride;
  float n = 0.0f, m[8] = {}, q[8] = {};
  if (p.eight < p.eights)
    gather<EIGHTS>(x, p.px * a.stride, (unsigned)(many - p.slot + p.px - 1) / (unsigned)p.px, at, a.c, n, m, q);
  float2 *out = a.part + (long)blockIdx.x * a.groups;
  by_group(s, p, n, m, q, a.c, a.c / a.groups, [&](int g, float mean, float squares) { out[g] = {mean, squares}; });
}

// A lane's eight channels' way from x to y.
struct Line {
  float mean[8], gain[8], bias[8];
  // First gamma and beta, so that their loads are under way early, then the statistics.
  __device__ __forceinline__ Line(const NormArgs &a, int c0, int at) {
#pragma unroll
    for (int i = 0; i < 8; i++) gain[i] = 1.0f, bias[i] = 0.0f;
    auto get = [&](const float *from, float *to) {
      const Eight<float> v = load_eight<false>(from + c0, at, a.span);
#pragma unroll
      for (int i = 0; i < 8; i++) to[i] = v[i];
    };
    if (a.gamma) get(a.gamma, gain);
    if (a.beta) get(a.beta, bias);
  }
  __device__ __forceinline__ void set(const NormArgs &a, int at, const float2 *stats) {
    const int per = a.c / a.groups;
    int g = at / per, in = at - g * per;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float2 st = stats[min(g, a.span / per - 1)];
      mean[i] = st.x;
      gain[i] *= st.y;
      if (++in == per) in = 0, g++;
    }
  }
};

// Eight results of pixel r from channel c0 + at on (`at` within the span).
template <typename Y, bool EIGHTS, int ACT>
__device__ __forceinline__ void put(const NormArgs &a, const Line &l, long r, int c0, int at, float *v) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = act8<ACT>((v[i] - l.mean[i]) * l.gain[i] + l.bias[i]);
  if constexpr (sizeof(Y) == 1) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (at + i >= a.span) v[i] = 0.0f;
      top = fmaxf(top, finite_magnitude(v[i]));
    }
    const int e = exponent8(max16(top));
    *(int2v *)((uint8_t *)a.y + r * a.ystride + c0 + at) = pack8(v, inverse_power(e));
    if ((at & 127) == 0) a.scales[r * a.scale_stride + (c0 + at) / 128] = (uint8_t)(e + 127);
  } else {
    Y *y = (Y *)a.y + r * a.ystride + c0;
    if (EIGHTS || at + 8 <= a.span)
      stream8(y + at, v);
    else
      store8<Y, false>(y, at, a.span, v);
  }
}

// A lane's `count` pixels r, r + px, ... from x on, `step` apart, from the last:
// a batch is loaded while the one after it (the first one by the caller) is written.
template <bool EIGHTS, typename T>
constexpr int BATCH = (sizeof(T) == 2 ? 4 : 2) / (EIGHTS ? 1 : 2);
template <bool EIGHTS, typename T>
__device__ __forceinline__ void load_batch(const T *x, Eight<T> (&to)[BATCH<EIGHTS, T>], long step, int k, int count,
                                           int at, int c) {
#pragma unroll
  for (int u = 0; u < BATCH<EIGHTS, T>; u++) to[u] = load_eight<EIGHTS>(x + max(min(k + u, count - 1), 0) * step, at, c);
}
template <bool EIGHTS, typename T>
__device__ __forceinline__ int last_batch(int count) {
  return (count - 1) / BATCH<EIGHTS, T> * BATCH<EIGHTS, T>;
}
template <bool EIGHTS, typename T, typename Y>
__device__ __forceinline__ void apply(const NormArgs &a, const Line &l, Eight<T> (&now)[BATCH<EIGHTS, T>], const T *x, long step,
                                      int count, long r, int px, int c0, int at) {
  constexpr int U = BATCH<EIGHTS, T>;
  with_act8(a.act, [&](auto act) {
    for (int k = last_batch<EIGHTS, T>(count); k >= 0; k -= U) {
      Eight<T> next[U];
      load_batch<EIGHTS>(x, next, step, k - U, count, at, a.span);
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)now[u][i];
        if (k + u < count) put<Y, EIGHTS, decltype(act)::value>(a, l, r + (long)(k + u) * px, c0, at, v);
      }
#pragma unroll
      for (int u = 0; u < U; u++) now[u] = next[u];
    }
  });
}

// The parts' statistics joined, and the same part of the pixels again, from its
// end.  The parts' means are summed from the first one's on, then the squares
// about their mean; all but the last part hold a.chunk pixels.  A lane may have
// some hundred parts to sum (one a group, where there are thousands), in f64: one
// after the other in f32 they left means 2e-6 of a deviation off.
template <typename T, typename Y, bool EIGHTS>
__global__ __launch_bounds__(LANES) void k_norm_apply(NormArgs a) {
  constexpr int HERE = 16;  // parts a lane keeps for the second sum
  extern __shared__ float lds[];
  const int lanes = blockDim.x;
  float *sums = lds, *means = lds + lanes;
  float2 *stats = (float2 *)(means + lanes);  // [group]: mean, 1 / deviation
  const int t = threadIdx.x, per = a.c / a.groups, image = blockIdx.x / a.chunks, mine = blockIdx.x % a.chunks;
  const Place p(a.c, sizeof(Y) == 1 ? 16 : 1, 0);
  const int at = p.eight * 8;
  const long begin = mine * a.chunk, r0 = image * a.pixels + begin + p.slot, step = p.px * a.stride;
  const T *x = (const T *)a.x + r0 * a.stride;
  const int count =
      p.eight < p.eights ? (unsigned)((int)min(a.chunk, a.pixels - begin) - p.slot + p.px - 1) / (unsigned)p.px : 0;
  Eight<T> now[BATCH<EIGHTS, T>];
  if (count > 0) load_batch<EIGHTS>(x, now, step, last_batch<EIGHTS, T>(count), count, at, a.c);
  Line l(a, 0, at);

  const float whole = (float)a.chunk, last = (float)(a.pixels - (a.chunks - 1) * a.chunk);
  for (int g0 = 0; g0 < a.groups; g0 += lanes) {
    const int many = min(a.groups - g0, lanes), rows = lanes / many, row = t / many, g = t - row * many;
    const float2 *part = a.part + (long)image * a.chunks * a.groups + g0 + g;
    const float base = part[0].x;
    // A lane's parts row, row + rows, ...: f(its mean and squares, its pixels).
    float2 v[HERE];
#pragma unroll
    for (int i = 0; i < HERE; i++)
      if (i * rows < a.chunks) v[i] = part[(long)min(row + i * rows, a.chunks - 1) * a.groups];
    auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < HERE; i++) {
        const int k = row + i * rows;
        if (i * rows < a.chunks) f(v[i], k >= a.chunks ? 0.0f : k == a.chunks - 1 ? last : whole);
      }
      for (int k = row + HERE * rows; k < a.chunks; k += rows) f(part[(long)k * a.groups], k == a.chunks - 1 ? last : whole);
    };
    auto sum = [&](float s) {  // over a group's lanes, in the first one
      __syncthreads();
      sums[t] = s;
      __syncthreads();
      int width = 1;
      while (width * 2 < rows) width *= 2;
      for (; width >= 16; width /= 2) {  // (halved down to 16, then one lane's sum)
        if (row < width && row + width < rows) sums[t] = s += sums[t + width * many];
        __syncthreads();
      }
      s = 0.0f;
      if (row == 0)
#pragma unroll 8
        for (int k = 0; k < min(rows, 16); k++) s += sums[k * many + t];
      return s;
    };
    double own = 0.0;
    if (row < rows) each([&](float2 x, float n) { own += n * (x.x - base); });
    float s = sum((float)own);
    if (row == 0) means[t] = base + s / (float)a.pixels;
    __syncthreads();
    const float mean = means[g];
    own = 0.0;
    if (row < rows)
      each([&](float2 x, float n) {
        const float d = x.x - mean;
        own += n > 0.0f ? x.y + (n * per) * d * d : 0.0f;
      });
    s = sum((float)own);
    if (row == 0) stats[g0 + t] = {mean, 1.0f / sqrtf(s / ((float)a.pixels * per) + a.eps)};
    __syncthreads();
  }

  if (count <= 0) return;
  l.set(a, at, stats);
  apply<EIGHTS, T, Y>(a, l, now, x, step, count, r0, p.px, 0, at);
}

// One launch: a workgroup a span of whole groups (and blocks of 128 channels)
// of an image, a.px lanes an eight whatever the span (so that the statistics do
// not depend on it).
template <typename T, typename Y, bool EIGHTS>
__global__ __launch_bounds__(LANES) void k_norm_one(NormArgs a) {
  extern __shared__ float lds[];
  const Shared s(lds);
  float2 *stats = (float2 *)(lds + 17 * blockDim.x);
  const Place p(a.span, sizeof(Y) == 1 ? 16 : 1, a.px);
  const int spans = a.c / a.span, image = blockIdx.x / spans, c0 = blockIdx.x % spans * a.span, at = p.eight * 8;
  const int per = a.c / a.groups;
  const long r0 = image * a.pixels + p.slot;
  const T *x = (const T *)a.x + r0 * a.stride + c0;
  const int count = p.eight < p.eights ? (unsigned)((int)a.pixels - p.slot + p.px - 1) / (unsigned)p.px : 0;
  float n = 0.0f, m[8] = {}, q[8] = {};
  Eight<T> now[BATCH<EIGHTS, T>];
  Line l(a, c0, at);
  if (count > 0) {
    gather<EIGHTS>(x, p.px * a.stride, count, at, a.span, n, m, q);
    load_batch<EIGHTS>(x, now, p.px * a.stride, last_batch<EIGHTS, T>(count), count, at, a.span);
  }
  by_group(s, p, n, m, q, a.span, per, [&](int g, float mean, float squares) {
    stats[g] = {mean, 1.0f / sqrtf(squares / ((float)a.pixels * per) + a.eps)};
  });
  __syncthreads();
  if (count == 0) return;
  l.set(a, at, stats);
  apply<EIGHTS, T, Y>(a, l, now, x, p.px * a.stride, count, r0, p.px, c0, at);
}

// The smallest run of whole groups and multiples of `unit` channels that c is made of.
int smallest_span(int c, int per, int unit) {
  int span = per;
  while (span % unit != 0 && span < c) span += per;
  return span % unit == 0 && c % span == 0 ? span : c;
}

ien_status run(ien_ctx *ctx, NormArgs a, long images, ien_out_type type, int y_bytes) {
  const int per = a.c / a.groups;
  const NormPlan plan = norm_plan(ctx->cus, (long)ctx->splitk_floats, images, a.pixels, a.c, a.groups, y_bytes);
  a.span = (int)plan.span;
  a.px = (int)plan.px;
  a.chunks = (int)plan.chunks;
  a.chunk = plan.chunk;
  a.part = (float2 *)ctx->splitk;
  const int lanes = (int)plan.lanes;
  const void *x = a.x;
  uint8_t *y = (uint8_t *)a.y, *scales = a.scales;
  auto go_eights = [&](auto t, auto u, auto e, long many) {
    using T = decltype(t);
    using Y = decltype(u);
    constexpr bool E = decltype(e)::value;
    const dim3 grid((unsigned)(many * plan.groups));
    if (plan.one) {
      const size_t shared = shared_floats(lanes) * 4 + a.span / per * sizeof(float2);
      hipLaunchKernelGGL((k_norm_one<T, Y, E>), grid, dim3(lanes), shared, ctx->stream, a);
    } else {
      hipLaunchKernelGGL((k_norm_stats<T, E>), grid, dim3(lanes), shared_floats(lanes) * 4, ctx->stream, a);
      hipLaunchKernelGGL((k_norm_apply<T, Y, E>), grid, dim3(lanes), 2 * lanes * 4 + a.groups * sizeof(float2), ctx->stream, a);
    }
  };
  const bool in_eights = a.c % 8 == 0;
  auto go = [&](auto t, auto u, long many) {
    in_eights ? go_eights(t, u, Act<1>{}, many) : go_eights(t, u, Act<0>{}, many);
  };
  const int x_bytes = type == IEN_OUT_F16 ? 2 : 4;
  for (long i = 0; i < images; i += plan.images) {  // (one turn but for a great many images)
    const long many = std::min(plan.images, images - i), r = i * a.pixels;
    a.x = (const uint8_t *)x + r * a.stride * x_bytes;
    a.y = y + r * a.ystride * y_bytes;
    a.scales = scales + r * a.scale_stride;
    if (x_bytes == 2)
      y_bytes == 1 ? go((_Float16)0, (uint8_t)0, many)
                   : y_bytes == 2 ? go((_Float16)0, (_Float16)0, many) : go((_Float16)0, 0.0f, many);
    else
      y_bytes == 1 ? go(0.0f, (uint8_t)0, many) : y_bytes == 2 ? go(0.0f, (_Float16)0, many) : go(0.0f, 0.0f, many);
  }
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

// What both entry points refuse, and the arguments they share.
ien_status describe(ien_ctx *ctx, const void *d_x, ien_out_type type, size_t images, size_t pixels, size_t c,
                    size_t stride, size_t groups, const float *d_gamma, const float *d_beta, float eps, ien_act act,
                    NormArgs *a) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  IEN_CHECK(type == IEN_OUT_F16 || type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)type);
  IEN_CHECK(act8_known(act), IEN_ERR_INPUT, "group norm takes no activation %d", (int)act);
  IEN_CHECK(c >= 1 && c <= 8192 && groups >= 1 && c % groups == 0, IEN_ERR_INPUT, "%zu channels in %zu groups", c,
            groups);
  IEN_CHECK(eps >= 0.0f && eps < 1e30f, IEN_ERR_INPUT, "eps %g", eps);
  IEN_CHECK(images < (1u << 20) && pixels < (1ull << 40) && stride < (1ull << 31), IEN_ERR_INPUT,
            "%zu maps of %zu pixels, %zu apart", images, pixels, stride);
  *a = NormArgs{};
  a->x = d_x;
  a->pixels = (long)pixels;
  a->stride = (long)stride;
  a->c = (int)c;
  a->groups = (int)groups;
  a->act = act;
  a->gamma = d_gamma;
  a->beta = d_beta;
  a->eps = eps;
  return IEN_OK;
}

}  // namespace

NormPlan norm_plan(int cus, long workspace, long images, long pixels, int c, int groups, int y_bytes) {
  NormPlan p{};
  const int per = c / groups;
  // One launch where a lane's share is a few pixels.
  const int wide = smallest_span(c, per, 128);
  p.px = std::min(64, LANES / ((wide + 127) / 128 * 16));
  p.one = pixels <= 8 * p.px;
  p.span = !p.one ? c : y_bytes == 1 ? wide : smallest_span(c, per, 8);
  const long eights = (p.span + 7) / 8;
  if (p.one) {
    p.lanes = ((y_bytes == 1 ? (eights + 15) / 16 * 16 : eights) * p.px + 63) / 64 * 64;
    p.chunks = 1;
    p.chunk = pixels;
    p.groups = c / p.span;
  } else {
    // A workgroup a part of at least four rounds of pixels, one for each CU where there
    // are as many (one for every other CU: 64 x 96 x 640 14.4 -> 15.2 us, into 8
    // bits 15.3 -> 17.2, 128 x 128 x 512 16.1 -> 19.2; 64 x 64 x 512, which has 128, 12.9).
    p.lanes = eights <= 512 ? 512 : LANES;
    const long px = p.lanes / eights, rounds = (pixels + px - 1) / px;
    const long parts = std::max(1L, std::min((rounds + 3) / 4, cus / images));
    p.chunk = std::min((rounds + parts - 1) / parts, (1L << 30) / px) * px;  // (counted in 32 bits)
    p.chunks = (pixels + p.chunk - 1) / p.chunk;
    p.groups = p.chunks;
  }
  const long fit = p.one ? images : workspace / 2 / (p.chunks * groups);
  p.images = std::max(1L, std::min({images, fit, (1L << 31) / (p.groups * p.lanes)}));
  return p;
}

}  // namespace ien

using namespace ien;

extern "C" {

ien_status ien_group_norm(ien_ctx *ctx, const void *d_x, ien_out_type type, size_t images, size_t pixels, size_t c,
                          size_t stride, size_t groups, const float *d_gamma, const float *d_beta, float eps,
                          ien_act act, void *d_y, ien_out_type y_type, size_t y_stride) {
  NormArgs a;
  const ien_status s = describe(ctx, d_x, type, images, pixels, c, stride, groups, d_gamma, d_beta, eps, act, &a);
  if (s != IEN_OK) return s;
  IEN_CHECK(y_type == IEN_OUT_F16 || y_type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)y_type);
  if (images == 0 || pixels == 0) return IEN_OK;
  IEN_CHECK(d_x && d_y && stride >= c && y_stride >= c && y_stride < (1ull << 31), IEN_ERR_INPUT,
            "no map, or pixels %zu and %zu apart for %zu channels", stride, y_stride, c);
  IEN_CHECK(d_x != d_y || (type == y_type && stride == y_stride), IEN_ERR_INPUT,
            "in place with another type or stride");
  a.y = d_y;
  a.ystride = (long)y_stride;
  return run(ctx, a, (long)images, type, y_type == IEN_OUT_F16 ? 2 : 4);
}

ien_status ien_group_norm8(ien_ctx *ctx, const void *d_x, ien_out_type type, size_t images, size_t pixels, size_t c,
                           size_t stride, size_t groups, const float *d_gamma, const float *d_beta, float eps,
                           ien_act act, const ien_rows8 *out) {
  NormArgs a;
  ien_status s = describe(ctx, d_x, type, images, pixels, c, stride, groups, d_gamma, d_beta, eps, act, &a);
  if (s != IEN_OK) return s;
  if (images == 0 || pixels == 0) return IEN_OK;
  IEN_CHECK(d_x && stride >= c, IEN_ERR_INPUT, "no map, or pixels %zu apart for %zu channels", stride, c);
  s = check_rows8(out, c, "group_norm8");
  if (s != IEN_OK) return s;
  a.y = out->data;
  a.ystride = (long)out->stride;
  a.scales = out->scales;
  a.scale_stride = (long)out->scale_stride;
  return run(ctx, a, (long)images, type, 1);
}

}  // extern "C"
