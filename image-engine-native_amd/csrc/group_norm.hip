// group_norm.hip -- group norm with an activation over channels-last maps
// (ien_group_norm, ien_group_norm8): y = act((x - m) / sqrt(v + eps) gamma +
// beta) with m and v over a map's pixels and a group's channels.

#include "eight_bits.h"

namespace ien {
namespace {

struct NormArgs {
  const void *x;
  long images, pixels, stride;
  int c, groups, act;
  const float *gamma, *beta;
  float eps;
  void *y;
  long ystride;
  uint8_t *scales;
  long scale_stride;
};

template <int N>
__device__ float block_sum(float v, float *lds) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N / 64; i++) s += lds[i];
  return s;
}

// A workgroup an image and group: the mean, then the squares of the
// deviations from it.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_stats(NormArgs a, float *__restrict__ stats) {
  __shared__ float lds[4];
  const int per = a.c / a.groups;
  const long image = blockIdx.x / a.groups, g = blockIdx.x % a.groups, n = a.pixels * per;
  const T *x = (const T *)a.x + image * a.pixels * a.stride + g * per;
  float s = 0.0f;
  for (long i = threadIdx.x; i < n; i += 256) s += (float)x[i / per * a.stride + i % per];
  const float mean = block_sum<256>(s, lds) / (float)n;
  s = 0.0f;
  for (long i = threadIdx.x; i < n; i += 256) {
    const float d = (float)x[i / per * a.stride + i % per] - mean;
    s += d * d;
  }
  const float var = block_sum<256>(s, lds) / (float)n;
  if (threadIdx.x == 0) {
    stats[2 * blockIdx.x] = mean;
    stats[2 * blockIdx.x + 1] = 1.0f / sqrtf(var + a.eps);
  }
}

// 16 lanes a block of 128 channels of a pixel.
template <typename T, typename Y>
__global__ __launch_bounds__(256) void k_norm_apply(NormArgs a, const float *__restrict__ stats) {
  const int blocks = (a.c + 127) / 128, per = a.c / a.groups;
  const long total = a.images * a.pixels * blocks;
  const int lane8 = (threadIdx.x & 15) * 8;
  for (long item = (long)blockIdx.x * 16 + threadIdx.x / 16; item < total; item += (long)gridDim.x * 16) {
    const long r = item / blocks, image = r / a.pixels;
    const int b = (int)(item - r * blocks), at = b * 128 + lane8;
    float v[8];
    load8<T, false>((const T *)a.x + r * a.stride, at, a.c, v);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int ch = at + i;
      if (ch < a.c) {
        const float *st = stats + 2 * (image * a.groups + ch / per);
        v[i] = (v[i] - st[0]) * st[1] * (a.gamma ? a.gamma[ch] : 1.0f) + (a.beta ? a.beta[ch] : 0.0f);
      }
    }
    with_act8(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (at + i < a.c) v[i] = act8<decltype(act)::value>(v[i]);
    });
    if constexpr (sizeof(Y) == 1) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) m = fmaxf(m, finite_magnitude(v[i]));
      const int e = exponent8(max16(m));
      *(int2v *)((uint8_t *)a.y + r * a.ystride + at) = pack8(v, inverse_power(e));
      if (lane8 == 0) a.scales[r * a.scale_stride + b] = (uint8_t)(e + 127);
    } else {
      store8<Y, false>((Y *)a.y + r * a.ystride, at, a.c, v);
    }
  }
}

ien_status run(ien_ctx *ctx, const NormArgs &a, ien_out_type type, int y_bytes) {
  IEN_CHECK(a.images * a.groups * 2 <= (long)ctx->splitk_floats, IEN_ERR_INPUT, "%ld maps of %d groups past the workspace",
            a.images, a.groups);
  const unsigned stat = (unsigned)(a.images * a.groups);
  const long items = a.images * a.pixels * ((a.c + 127) / 128);
  const unsigned grid = (unsigned)std::min((items + 15) / 16, 1L << 24);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL(k_norm_stats<T>, dim3(stat), dim3(256), 0, ctx->stream, a, ctx->splitk);
    if (y_bytes == 1)
      hipLaunchKernelGGL((k_norm_apply<T, uint8_t>), dim3(grid), dim3(256), 0, ctx->stream, a, ctx->splitk);
    else if (y_bytes == 2)
      hipLaunchKernelGGL((k_norm_apply<T, _Float16>), dim3(grid), dim3(256), 0, ctx->stream, a, ctx->splitk);
    else
      hipLaunchKernelGGL((k_norm_apply<T, float>), dim3(grid), dim3(256), 0, ctx->stream, a, ctx->splitk);
  };
  type == IEN_OUT_F16 ? go((_Float16)0) : go(0.0f);
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
  a->images = (long)images;
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
  return run(ctx, a, type, y_type == IEN_OUT_F16 ? 2 : 4);
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
  return run(ctx, a, type, 1);
}

}  // extern "C"
