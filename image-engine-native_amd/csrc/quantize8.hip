// quantize8.hip -- rows in 8 bits: blocks of 128 e4m3 values under a
// power-of-two scale, written and read back (ien_quantize8, ien_dequantize8),
// and the weights of ien_multiply8 (ien_matrix8_new).
//
// The mathematics is a maximum over 128 values, an exponent taken from its
// bits, a product with a power of two (exact) and one rounding, so the passes
// are bound by memory.  16 lanes hold a block, 8 values (one 16-byte load of
// f16) each, and reduce the maximum by lane moves inside a row of 16; a wave
// takes four blocks at once.  EIGHTS: k is in eights.  98304 rows of 512 f32
// values written and read back: 97 us, 4.1 TB/s of the f32 values alone and 5.2
// with the bytes between.

#include <algorithm>
#include <new>

#include "eight_bits.h"

namespace ien {

ien_status check_rows8(const ien_rows8 *r, size_t k, const char *what) {
  IEN_CHECK(r && r->data && r->scales, IEN_ERR_INPUT, "%s: no rows in 8 bits", what);
  IEN_CHECK(((uintptr_t)r->data & 15) == 0 && ((uintptr_t)r->scales & 3) == 0, IEN_ERR_INPUT,
            "%s: rows in 8 bits unaligned", what);
  IEN_CHECK(r->stride % 16 == 0 && r->stride >= ien_rows8_stride(k) && r->scale_stride % 4 == 0 &&
                r->scale_stride >= ien_rows8_scale_stride(k),
            IEN_ERR_INPUT, "%s: strides %zu and %zu for rows of %zu", what, r->stride, r->scale_stride, k);
  return IEN_OK;
}

namespace {

struct Rows8Args {
  uint8_t *data;
  long stride;
  uint8_t *scales;
  long scale_stride;
};
Rows8Args args_of(const ien_rows8 &r) { return {r.data, (long)r.stride, r.scales, (long)r.scale_stride}; }

constexpr int ITEMS = 16;  // blocks a workgroup of 256 lanes takes at a time

template <typename T, bool EIGHTS>
__global__ __launch_bounds__(256) void k_quantize8(const T *__restrict__ x, long stride, long rows, long k, int blocks,
                                                   Rows8Args q) {
  const long total = rows * blocks, lane8 = (threadIdx.x & 15) * 8;
  for (long item = (long)blockIdx.x * ITEMS + threadIdx.x / 16; item < total; item += (long)gridDim.x * ITEMS) {
    const long r = item / blocks;
    const int b = (int)(item - r * blocks);
    const long at = (long)b * BLOCK8 + lane8;
    float v[8] = {};
    if (at + 8 <= k)
      load8<T, true>(x + r * stride, at, k, v);
    else if (!EIGHTS)
      load8<T, false>(x + r * stride, at, k, v);
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, finite_magnitude(v[i]));
    const int e = exponent8(max16(m));
    *(int2v *)(q.data + r * q.stride + at) = pack8(v, inverse_power(e));
    if (lane8 == 0) q.scales[r * q.scale_stride + b] = (uint8_t)(e + 127);
  }
}

template <typename T, bool EIGHTS>
__global__ __launch_bounds__(256) void k_dequantize8(Rows8Args q, long rows, long k, int blocks, T *__restrict__ y,
                                                     long stride) {
  const long total = rows * blocks, lane8 = (threadIdx.x & 15) * 8;
  for (long item = (long)blockIdx.x * ITEMS + threadIdx.x / 16; item < total; item += (long)gridDim.x * ITEMS) {
    const long r = item / blocks;
    const int b = (int)(item - r * blocks);
    const long at = (long)b * BLOCK8 + lane8;
    if (at >= k) continue;
    const int2v p = *(const int2v *)(q.data + r * q.stride + at);
    const float s = scale_power(q.scales[r * q.scale_stride + b]);
    const float v[8] = {
        s * __builtin_amdgcn_cvt_f32_fp8(p.x, 0), s * __builtin_amdgcn_cvt_f32_fp8(p.x, 1),
        s * __builtin_amdgcn_cvt_f32_fp8(p.x, 2), s * __builtin_amdgcn_cvt_f32_fp8(p.x, 3),
        s * __builtin_amdgcn_cvt_f32_fp8(p.y, 0), s * __builtin_amdgcn_cvt_f32_fp8(p.y, 1),
        s * __builtin_amdgcn_cvt_f32_fp8(p.y, 2), s * __builtin_amdgcn_cvt_f32_fp8(p.y, 3)};
    if (EIGHTS || at + 8 <= k)
      stream8(y + r * stride + at, v);
    else
      store8<T, false>(y + r * stride, at, k, v);
  }
}

// A thread an output and panel: the maximum over the panel's channels, then
// the bytes (neighbouring threads read neighbouring outputs' weights).
template <typename T>
__global__ __launch_bounds__(256) void k_pack8(const T *__restrict__ w, int c, long n, long npad, int cb,
                                               uint8_t *__restrict__ out, uint32_t *__restrict__ scales) {
  const long o = (long)blockIdx.x * 256 + threadIdx.x;
  if (o >= npad) return;
  const int panel = blockIdx.y, t = panel / cb, c0 = (panel - t * cb) * BLOCK8, cn = min(BLOCK8, c - c0);
  const T *src = w + ((long)t * c + c0) * n + o;
  float m = 0.0f;
  if (o < n)
    for (int i = 0; i < cn; i++) m = fmaxf(m, finite_magnitude((float)src[i * n]));
  const int e = exponent8(m);
  const float inv = inverse_power(e);
  uint8_t *dst = out + ((long)panel * npad + o) * BLOCK8;
  for (int i = 0; i < BLOCK8; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = o < n && i + j < cn ? (float)src[(i + j) * n] : 0.0f;
    *(int2v *)(dst + i) = pack8(v, inv);
  }
  scales[(long)panel * npad + o] = (uint32_t)(e + 127);
}

}  // namespace

// (A launch counts its lanes in 32 bits: at most 2^28 of them, which take turns.)
unsigned quantize8_grid(long blocks) { return (unsigned)std::min((blocks + ITEMS - 1) / ITEMS, 1L << 20); }

}  // namespace ien

using namespace ien;

extern "C" {

size_t ien_rows8_stride(size_t k) { return BLOCK8 * blocks8(k); }
size_t ien_rows8_scale_stride(size_t k) { return 4 * ((blocks8(k) + 3) / 4); }

ien_status ien_quantize8(ien_ctx *ctx, const void *d_x, ien_out_type type, size_t rows, size_t k, size_t stride,
                         const ien_rows8 *out) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  IEN_CHECK(type == IEN_OUT_F16 || type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)type);
  IEN_CHECK(k < (1u << 30) && rows < (1ull << 40), IEN_ERR_INPUT, "%zu rows of %zu", rows, k);
  if (rows == 0 || k == 0) return IEN_OK;
  IEN_CHECK(d_x && stride >= k, IEN_ERR_INPUT, "no rows, or %zu apart for k = %zu", stride, k);
  const ien_status s = check_rows8(out, k, "quantize8");
  if (s != IEN_OK) return s;
  const int blocks = (int)blocks8(k);
  const dim3 grid(quantize8_grid((long)rows * blocks));
  const bool eights = k % 8 == 0;
  auto launch = [&](auto kernel, auto *x) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, x, (long)stride, (long)rows, (long)k, blocks,
                       args_of(*out));
  };
  if (type == IEN_OUT_F16)
    eights ? launch(k_quantize8<_Float16, true>, (const _Float16 *)d_x)
        : launch(k_quantize8<_Float16, false>, (const _Float16 *)d_x);
  else
    eights ? launch(k_quantize8<float, true>, (const float *)d_x) : launch(k_quantize8<float, false>, (const float *)d_x);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

ien_status ien_dequantize8(ien_ctx *ctx, const ien_rows8 *x, size_t rows, size_t k, void *d_y, ien_out_type type,
                           size_t stride) {
  IEN_CHECK(ctx, IEN_ERR_INPUT, "no context");
  IEN_CHECK(type == IEN_OUT_F16 || type == IEN_OUT_F32, IEN_ERR_INPUT, "type %d", (int)type);
  IEN_CHECK(k < (1u << 30) && rows < (1ull << 40), IEN_ERR_INPUT, "%zu rows of %zu", rows, k);
  if (rows == 0 || k == 0) return IEN_OK;
  IEN_CHECK(d_y && stride >= k, IEN_ERR_INPUT, "no rows, or %zu apart for k = %zu", stride, k);
  const ien_status s = check_rows8(x, k, "dequantize8");
  if (s != IEN_OK) return s;
  const int blocks = (int)blocks8(k);
  const dim3 grid(quantize8_grid((long)rows * blocks));
  const bool eights = k % 8 == 0;
  auto launch = [&](auto kernel, auto *y) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, args_of(*x), (long)rows, (long)k, blocks, y,
                       (long)stride);
  };
  if (type == IEN_OUT_F16)
    eights ? launch(k_dequantize8<_Float16, true>, (_Float16 *)d_y) : launch(k_dequantize8<_Float16, false>, (_Float16 *)d_y);
  else
    eights ? launch(k_dequantize8<float, true>, (float *)d_y) : launch(k_dequantize8<float, false>, (float *)d_y);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

ien_status ien_matrix8_new(ien_ctx *ctx, const void *w, ien_wtype wtype, size_t taps, size_t c, size_t n,
                           const float *bias, ien_matrix8 **out) {
  IEN_CHECK(ctx && w && out, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(wtype == IEN_W_F32 || wtype == IEN_W_F16, IEN_ERR_INPUT, "weight type %d", (int)wtype);
  IEN_CHECK((taps == 1 || taps == 9) && c > 0 && n > 0 && c < (1u << 22) && n < (1u << 22) && taps * blocks8(c) < 65536,
            IEN_ERR_INPUT, "weights of %zu taps x %zu x %zu", taps, c, n);
  ien_matrix8 *m = new (std::nothrow) ien_matrix8;
  IEN_CHECK(m, IEN_ERR_GPU, "8-bit weights: out of host memory");
  m->ctx = ctx;
  m->taps = taps;
  m->c = c;
  m->n = n;
  m->cb = (int)blocks8(c);
  m->npad = (long)((n + 127) / 128 * 128);
  const size_t panels = taps * m->cb, bytes = taps * c * n * (wtype == IEN_W_F16 ? 2 : 4);
  void *raw = nullptr;
  hipError_t e = hipSetDevice(ctx->device);
  if (e == hipSuccess) e = hipMalloc(&raw, bytes);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_w, ((panels + SLACK8) * m->npad + 128) * BLOCK8);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_scales, ((panels + SLACK8) * m->npad + 128) * 4);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_bias, m->npad * 4);
  if (e == hipSuccess) e = hipMemcpyAsync(raw, w, bytes, hipMemcpyHostToDevice, ctx->stream);
  if (e == hipSuccess) e = hipMemsetAsync(m->d_bias, 0, m->npad * 4, ctx->stream);
  if (e == hipSuccess && bias) e = hipMemcpyAsync(m->d_bias, bias, n * 4, hipMemcpyHostToDevice, ctx->stream);
  if (e == hipSuccess) {
    const dim3 grid((unsigned)((m->npad + 255) / 256), (unsigned)panels);
    if (wtype == IEN_W_F16)
      hipLaunchKernelGGL(k_pack8<_Float16>, grid, dim3(256), 0, ctx->stream, (const _Float16 *)raw, (int)c, (long)n,
                         m->npad, m->cb, m->d_w, m->d_scales);
    else
      hipLaunchKernelGGL(k_pack8<float>, grid, dim3(256), 0, ctx->stream, (const float *)raw, (int)c, (long)n,
                         m->npad, m->cb, m->d_w, m->d_scales);
    e = hipGetLastError();
  }
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  (void)hipFree(raw);
  if (e != hipSuccess) {
    ien_matrix8_free(m);
    return fail(IEN_ERR_GPU, "8-bit weights: %s", hipGetErrorString(e));
  }
  *out = m;
  return IEN_OK;
}

void ien_matrix8_free(ien_matrix8 *m) {
  if (!m) return;
  if (m->ctx) (void)hipSetDevice(m->ctx->device);
  (void)hipFree(m->d_w);
  (void)hipFree(m->d_scales);
  (void)hipFree(m->d_bias);
  delete m;
}

}  // extern "C"
