// experts8.hip -- the experts' weights in 8 bits (ien_experts8_new): panels of
// 128 channels as ien_matrix8's, one expert after another.  A gated product's
// columns go in turns of 32 gates and the 32 they multiply, so that a lane of a
// matrix instruction's result holds both.

#include <new>

#include "experts.h"

namespace ien {
namespace {

// A thread a packed column and panel: the maximum over the panel's channels,
// then the bytes (neighbouring threads read neighbouring columns).
template <typename T>
__global__ __launch_bounds__(256) void k_pack_experts(const T *__restrict__ w, const float *__restrict__ bias, long c,
                                                      long n, int gated, long npad, int cb, uint8_t *__restrict__ out,
                                                      uint32_t *__restrict__ scales, float *__restrict__ biases) {
  const long o = (long)blockIdx.x * 256 + threadIdx.x;
  if (o >= npad) return;
  const int panel = blockIdx.y, expert = panel / cb, b = panel - expert * cb;
  const int cn = (int)min((long)BLOCK8, c - (long)b * BLOCK8);
  const long at = gated ? o / 64 * 32 + o % 32 : o, outs = gated ? n / 2 : n;
  const long column = at >= outs ? -1 : gated && o % 64 >= 32 ? outs + at : at;
  const T *src = w + (expert * c + (long)b * BLOCK8) * n + column;
  float m = 0.0f;
  if (column >= 0)
    for (int i = 0; i < cn; i++) m = fmaxf(m, finite_magnitude((float)src[i * n]));
  const int e = exponent8(m);
  const float inv = inverse_power(e);
  uint8_t *dst = out + ((long)panel * npad + o) * BLOCK8;
  for (int i = 0; i < BLOCK8; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = column >= 0 && i + j < cn ? (float)src[(i + j) * n] : 0.0f;
    *(int2v *)(dst + i) = pack8(v, inv);
  }
  scales[(long)panel * npad + o] = (uint32_t)(e + 127);
  if (b == 0) biases[expert * npad + o] = bias && column >= 0 ? bias[expert * n + column] : 0.0f;
}

}  // namespace
}  // namespace ien

using namespace ien;

extern "C" {

ien_status ien_experts8_new(ien_ctx *ctx, const void *d_w, ien_wtype wtype, size_t experts, size_t c, size_t n,
                            int gated, const float *d_bias, ien_experts8 **out) {
  IEN_CHECK(ctx && d_w && out, IEN_ERR_INPUT, "null argument");
  IEN_CHECK(wtype == IEN_W_F32 || wtype == IEN_W_F16, IEN_ERR_INPUT, "weight type %d", (int)wtype);
  IEN_CHECK(experts >= 1 && experts <= MAX_EXPERTS && c > 0 && n > 0 && c < (1u << 22) && n < (1u << 22) &&
                (!gated || n % 2 == 0) && experts * blocks8(c) < 65536,
            IEN_ERR_INPUT, "%s weights of %zu experts x %zu x %zu", gated ? "gated" : "plain", experts, c, n);
  const long npad = gated ? 2 * (long)((n / 2 + 127) / 128 * 128) : (long)((n + 127) / 128 * 128);
  const size_t panels = experts * blocks8(c);
  // (A tile addresses an expert's scales by 31-bit offsets.)
  IEN_CHECK(blocks8(c) * (size_t)npad < (1ull << 28), IEN_ERR_INPUT, "too many weights an expert: %zu x %zu", c, n);
  ien_experts8 *m = new (std::nothrow) ien_experts8;
  IEN_CHECK(m, IEN_ERR_GPU, "experts' weights: out of host memory");
  m->ctx = ctx;
  m->experts = experts;
  m->c = c;
  m->n = gated ? n / 2 : n;
  m->gated = gated != 0;
  m->cb = (int)blocks8(c);
  m->npad = npad;
  hipError_t e = hipSetDevice(ctx->device);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_w, ((panels + SLACK8) * npad + 128) * BLOCK8);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_scales, ((panels + SLACK8) * npad + 128) * 4);
  if (e == hipSuccess) e = hipMalloc((void **)&m->d_bias, experts * npad * 4);
  if (e == hipSuccess) {
    const dim3 grid((unsigned)((npad + 255) / 256), (unsigned)panels);
    if (wtype == IEN_W_F16)
      hipLaunchKernelGGL(k_pack_experts<_Float16>, grid, dim3(256), 0, ctx->stream, (const _Float16 *)d_w, d_bias,
                         (long)c, (long)n, m->gated, npad, m->cb, m->d_w, m->d_scales, m->d_bias);
    else
      hipLaunchKernelGGL(k_pack_experts<float>, grid, dim3(256), 0, ctx->stream, (const float *)d_w, d_bias, (long)c,
                         (long)n, m->gated, npad, m->cb, m->d_w, m->d_scales, m->d_bias);
    e = hipGetLastError();
  }
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    ien_experts8_free(m);
    return fail(IEN_ERR_GPU, "experts' weights: %s", hipGetErrorString(e));
  }
  *out = m;
  return IEN_OK;
}

void ien_experts8_free(ien_experts8 *m) {
  if (!m) return;
  if (m->ctx) (void)hipSetDevice(m->ctx->device);
  (void)hipFree(m->d_w);
  (void)hipFree(m->d_scales);
  (void)hipFree(m->d_bias);
  delete m;
}

}  // extern "C"
