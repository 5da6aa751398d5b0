// rms_norm.hip -- the sum of two maps' rows and its root-mean-square norm, in
// f16 or f32 and in 8 bits (ien_rms_norm):
//   s = x + add,  y = s / sqrt(mean(s^2) + eps) gamma
//
// A row is held in registers by 16, 64 or 256 lanes, up to four eights of
// channels each, so everything is read once and written once and memory bounds
// it.  The squares are added in f64: they neither overflow nor lose digits
// whatever the row holds, and two vector instructions a value are far below
// what the memory takes.  16 lanes' eights are a block of 128, whose scale they
// find among themselves.  65536 x 1024 in f16, sum and norm: 93 us, 5.8 TB/s;
// 16384 x 1536 with the norm in f16 and 8 bits 42 us, 5.4 TB/s.

#include <algorithm>
#include <type_traits>

#include "eight_bits.h"

namespace ien {
namespace {

struct RmsArgs {
  const void *x, *add;
  void *sum, *y;
  long stride, add_stride, sum_stride, y_stride;
  const float *gamma;
  uint8_t *data, *scales;
  long data_stride, scale_stride;
  long rows;
  int c, y_f32;
  float eps;
};

__device__ __forceinline__ double sum64(double v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  return v;
}

enum { NO_ADD, ADD_F16, ADD_F32 };

typedef float float8_any __attribute__((ext_vector_type(8), aligned(4)));
template <typename T>
struct Raw {
  typedef half8_any type;
};
template <>
struct Raw<float> {
  typedef float8_any type;
};

// Eight channels of a row as they are, past the last one anything.  EIGHTS: the row is
// whole eights; else its end is read one by one, that last one again past it (no branch
// between one load and the next, and nothing uses them yet).
template <bool EIGHTS, typename T>
__device__ __forceinline__ typename Raw<T>::type raw8(const T *row, int at, int c) {
  typename Raw<T>::type v;
  if constexpr (EIGHTS) v = (T)0.0f;
  if (at + 8 <= c) {
    v = *(const typename Raw<T>::type *)(row + at);
  } else if constexpr (!EIGHTS) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = row[min(at + i, c - 1)];
  }
  return v;
}

// L lanes a row, N eights of channels a lane: eight n of lane l is n L + l.  gamma is
// read first, for the rows that the workgroup takes one after another (behind them
// 16384 x 1536 takes 50 us in place of 42).  Rows of whole eights need no choice a
// channel: with one, vector instructions were 88 % of the cycles.
template <typename X, int ADD, int L, int N, bool EIGHTS>
__global__ __launch_bounds__(256) void k_rms_norm(RmsArgs a) {
  typedef std::conditional_t<ADD == ADD_F16, _Float16, float> A;
  constexpr int ROWS = 256 / L;
  __shared__ double part[4];
  const int lane = threadIdx.x % L, slot = threadIdx.x / L, c = a.c;
  const int padded = (c + BLOCK8 - 1) / BLOCK8 * BLOCK8;
  float g[N][8];
#pragma unroll
  for (int n = 0; n < N; n++) {
    const int at = 8 * (n * L + lane);
    float8_any v = 1.0f;
    if (a.gamma) v = raw8<EIGHTS>(a.gamma, at, c);
#pragma unroll
    for (int i = 0; i < 8; i++) g[n][i] = v[i];
  }
  for (long r0 = (long)blockIdx.x * ROWS; r0 < a.rows; r0 += (long)gridDim.x * ROWS) {
    const bool some = r0 + slot < a.rows;  // (all lanes stay: they find maxima and sums together)
    const long r = some ? r0 + slot : a.rows - 1;
    typename Raw<X>::type xs[N];
    typename Raw<A>::type as[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
      xs[n] = raw8<EIGHTS>((const X *)a.x + r * a.stride, 8 * (n * L + lane), c);
      if constexpr (ADD != NO_ADD) as[n] = raw8<EIGHTS>((const A *)a.add + r * a.add_stride, 8 * (n * L + lane), c);
    }
    float v[N][8];
    double squares = 0.0;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        v[n][i] = (float)xs[n][i];
        if constexpr (ADD != NO_ADD) v[n][i] += (float)as[n][i];
        if (!EIGHTS && 8 * (n * L + lane) + i >= c) v[n][i] = 0.0f;
        squares = fma((double)v[n][i], (double)v[n][i], squares);
      }
    if constexpr (L == 16) {
#pragma unroll
      for (int m = 1; m < 16; m *= 2) squares += __shfl_xor(squares, m);
    } else {
      squares = sum64(squares);
      if constexpr (L == 256) {
        __syncthreads();  // (the last row's parts are read)
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = squares;
        __syncthreads();
        squares = (part[0] + part[1]) + (part[2] + part[3]);
      }
    }
    // A root that is past what has a normal reciprocal in f32 (of f32 rows, and where it is small without an epsilon) is
    // taken towards 1 by a power of two, and so are the values that it divides.
    const double root = sqrt(squares / c + (double)a.eps);
    const float power = root < 0x1p-126 ? 0x1p64f : root > 0x1p126 ? 0x1p-64f : 1.0f;
    const float inv = (float)(1.0 / (root * (double)power));
    const bool far = (sizeof(X) == 4 || ADD == ADD_F32) && __ballot(power != 1.0f);
    auto store = [&](auto *row, int at, const float *w) {
      if (EIGHTS || at + 8 <= c)
        stream8(row + at, w);
      else
        store8<std::remove_reference_t<decltype(*row)>, false>(row, at, c, w);
    };
#pragma unroll
    for (int n = 0; n < N; n++) {
      const int at = 8 * (n * L + lane);
      if (a.sum && some && at < c) store((X *)a.sum + r * a.sum_stride, at, v[n]);
      if (far) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[n][i] *= power;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) v[n][i] = v[n][i] * inv * g[n][i];
      if (a.y && some && at < c) {
        if (a.y_f32)
          store((float *)a.y + r * a.y_stride, at, v[n]);
        else
          store((_Float16 *)a.y + r * a.y_stride, at, v[n]);
      }
      if (a.data) {
        if constexpr (!EIGHTS) {
#pragma unroll
          for (int i = 0; i < 8; i++) v[n][i] = at + i < c ? v[n][i] : 0.0f;
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[n][i]));  // (a NaN is passed over)
        if (__ballot(!finite8(m))) {  // infinities, which are NaN and no largest magnitude
          m = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            m = fmaxf(m, finite_magnitude(v[n][i]));
            if (!finite8(v[n][i])) v[n][i] = __uint_as_float(0x7fc00000);
          }
        }
        const int e = exponent8(max16(at < c ? m : 0.0f));
        const float unit = inverse_power(e);
        int2v p;
        p.x = __builtin_amdgcn_cvt_pk_fp8_f32(v[n][0] * unit, v[n][1] * unit, 0, false);
        p.x = __builtin_amdgcn_cvt_pk_fp8_f32(v[n][2] * unit, v[n][3] * unit, p.x, true);
        p.y = __builtin_amdgcn_cvt_pk_fp8_f32(v[n][4] * unit, v[n][5] * unit, 0, false);
        p.y = __builtin_amdgcn_cvt_pk_fp8_f32(v[n][6] * unit, v[n][7] * unit, p.y, true);
        if (some && at < padded) {
          *(int2v *)(a.data + r * a.data_stride + at) = at < c ? p : int2v{};
          if (at % BLOCK8 == 0) a.scales[r * a.scale_stride + at / BLOCK8] = (uint8_t)(e + 127);
        }
      }
    }
  }
}

template <typename X, int ADD, bool EIGHTS>
void launch_rows(ien_ctx *ctx, const RmsArgs &a) {
  // Workgroups take rows in turns, so many of them a CU (us, 8, 16, 32 and one for every four rows: 65536 x 1024
  // 98.0, 95.9, 93.0, 93.7; 100000 x 96 16.5, 15.8, 17.6, 17.8; 4000 x 8192 57.1, 60.5, 60.2, 60.1).  A wave a row up to
  // 2048 channels: a workgroup's barriers cost more than its lanes save (16384 x 1536 42.3 and 45.8 at best).
  auto go = [&](auto kernel, int rows, int many) {
    const dim3 grid((unsigned)std::min((a.rows + rows - 1) / rows, (long)many * ctx->cus));
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, a);
  };
  if (a.c <= 128) go(k_rms_norm<X, ADD, 16, 1, EIGHTS>, 16, 16);
  else if (a.c <= 512) go(k_rms_norm<X, ADD, 64, 1, EIGHTS>, 4, 32);
  else if (a.c <= 1024) go(k_rms_norm<X, ADD, 64, 2, EIGHTS>, 4, 32);
  else if (a.c <= 1536) go(k_rms_norm<X, ADD, 64, 3, EIGHTS>, 4, 32);
  else if (a.c <= 2048) go(k_rms_norm<X, ADD, 64, 4, EIGHTS>, 4, 32);
  else if (a.c <= 4096) go(k_rms_norm<X, ADD, 256, 2, EIGHTS>, 1, 8);
  else go(k_rms_norm<X, ADD, 256, 4, EIGHTS>, 1, 8);
}

template <typename X, int ADD>
void launch(ien_ctx *ctx, const RmsArgs &a) {
  a.c % 8 == 0 ? launch_rows<X, ADD, true>(ctx, a) : launch_rows<X, ADD, false>(ctx, a);
}

bool known(ien_out_type t) { return t == IEN_OUT_F16 || t == IEN_OUT_F32; }

}  // namespace
}  // namespace ien

using namespace ien;

extern "C" ien_status ien_rms_norm(ien_ctx *ctx, const void *d_x, ien_out_type type, size_t rows, size_t c,
                                   size_t stride, const void *d_add, ien_out_type add_type, size_t add_stride,
                                   void *d_sum, size_t sum_stride, const float *d_gamma, float eps, void *d_y,
                                   ien_out_type y_type, size_t y_stride, const ien_rows8 *out8) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  IEN_CHECK(known(type) && (!d_add || known(add_type)) && (!d_y || known(y_type)), IEN_ERR_INPUT,
            "rms_norm of types %d and %d into %d", (int)type, (int)add_type, (int)y_type);
  IEN_CHECK(c <= 8192 && rows < (1ull << 40), IEN_ERR_INPUT, "rms_norm of %zu rows of %zu", rows, c);
  IEN_CHECK(eps >= 0.0f, IEN_ERR_INPUT, "rms_norm with epsilon %g", (double)eps);
  if (rows == 0 || c == 0) return IEN_OK;
  IEN_CHECK(d_x && stride >= c && (!d_add || add_stride >= c) && (!d_sum || sum_stride >= c) && (!d_y || y_stride >= c),
            IEN_ERR_INPUT, "rms_norm: no rows, or %zu, %zu, %zu and %zu apart for c = %zu", stride, add_stride,
            sum_stride, y_stride, c);
  RmsArgs a{};
  if (out8) {
    const ien_status s = check_rows8(out8, c, "rms_norm");
    if (s != IEN_OK) return s;
    a.data = out8->data;
    a.scales = out8->scales;
    a.data_stride = (long)out8->stride;
    a.scale_stride = (long)out8->scale_stride;
  }
  a.x = d_x;
  a.add = d_add;
  a.sum = d_sum;
  a.y = d_y;
  a.stride = (long)stride;
  a.add_stride = (long)add_stride;
  a.sum_stride = (long)sum_stride;
  a.y_stride = (long)y_stride;
  a.gamma = d_gamma;
  a.rows = (long)rows;
  a.c = (int)c;
  a.y_f32 = y_type == IEN_OUT_F32;
  a.eps = eps;
  const int add = !d_add ? NO_ADD : add_type == IEN_OUT_F16 ? ADD_F16 : ADD_F32;
  if (type == IEN_OUT_F16) {
    if (add == NO_ADD) launch<_Float16, NO_ADD>(ctx, a);
    else if (add == ADD_F16) launch<_Float16, ADD_F16>(ctx, a);
    else launch<_Float16, ADD_F32>(ctx, a);
  } else {
    if (add == NO_ADD) launch<float, NO_ADD>(ctx, a);
    else if (add == ADD_F16) launch<float, ADD_F16>(ctx, a);
    else launch<float, ADD_F32>(ctx, a);
  }
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}
