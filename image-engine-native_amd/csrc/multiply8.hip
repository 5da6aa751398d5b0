// multiply8.hip -- products of rows in 8 bits with weights in 8 bits, plain
// rows and 3 x 3 convolutions (ien_multiply8), on the scaled 8-bit matrix
// instructions of gfx950:
//   y[r][n] = act(sum over blocks b of 2^(ex[r][b] + ew[b][n])
//                 sum over k in b of qx[r][k] qw[k][n] + bias[n] + add[r][n])
// v_mfma_scale_f32_32x32x64 takes a scale byte a row and 32 values of each
// operand; a block of 128 is two instructions under the same bytes, so the
// scales cost no vector instruction a product.
//
// The 8-bit instructions line the products of a few neighbouring values up on
// some 16 bits before they are added (measured: 2^16 + 1 inside one lane's
// values loses the 1; sums of 64 random products are off by 1.4e-5 of
// themselves, whatever their accumulator holds).  That is a fortieth of an f16
// output's own rounding, and as much as f32 outputs would be off in all.
// Those take their operands as bf16, which holds e4m3 values under any of the
// scales exactly, and the bf16 instructions (6e-9), at half the rate.

#include "eight_bits.h"

namespace ien {
namespace {

typedef int int8v __attribute__((ext_vector_type(8)));

struct Args8 {
  const uint8_t *x;
  long xs;
  const uint8_t *scales;
  long ss;
  int taps, cb, step;
  long images, H, W, OH, OW;  // rows: 1 map of 1 x rows
  long row0, rows;
  const uint8_t *w;
  const uint32_t *ws;
  const float *bias;
  long n, npad;
  void *y;
  long ys;
  int f32, act;
  const void *add;
  long as;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight e4m3 bytes under a scale as bf16.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A wave 32 rows x 32 outputs.  The weights are the A operand: a lane gets
// one row's results, four consecutive outputs at a time.
__global__ __launch_bounds__(256) void k_multiply8(Args8 a) {
  const int lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const long n0 = ((long)blockIdx.x * 4 + threadIdx.x / 64) * 32;
  if (n0 >= a.npad) return;
  const long r = (long)blockIdx.y * 32 + l32;
  const bool live = r < a.rows;
  const long p = a.row0 + (live ? r : 0), image = p / (a.OH * a.OW), q = p - image * a.OH * a.OW;
  const long oy = q / a.OW, ox = q - oy * a.OW;
  floatx16 acc = {};
  for (int t = 0; t < a.taps; t++) {
    const long iy = oy * a.step + (a.taps == 9 ? t / 3 - 1 : 0), ix = ox * a.step + (a.taps == 9 ? t % 3 - 1 : 0);
    const bool in = live && iy >= 0 && iy < a.H && ix >= 0 && ix < a.W;
    const long pixel = in ? (image * a.H + iy) * a.W + ix : 0;
    const uint8_t *x = a.x + pixel * a.xs;
    for (int b = 0; b < a.cb; b++) {
      const long panel = ((long)t * a.cb + b) * a.npad + n0 + l32;
      const int sx = in ? a.scales[pixel * a.ss + b] : 127, sw = (int)a.ws[panel];
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const int8v wv = *(const int8v *)(a.w + panel * 128 + s * 64 + hi * 32);
        int8v xv = {};
        if (in) {  // rows are 16-byte aligned only
          u32x4 lo = *(const u32x4 *)(x + b * 128 + s * 64 + hi * 32), up = *(const u32x4 *)(x + b * 128 + s * 64 + hi * 32 + 16);
          __builtin_memcpy(&xv, &lo, 16);
          __builtin_memcpy((char *)&xv + 16, &up, 16);
        }
        if (!a.f32) {
          acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, acc, 0, 0, 0, sw, 0, sx);
        } else {
          const float fw = scale_power(sw), fx = scale_power(sx);
#pragma unroll
          for (int i = 0; i < 8; i += 2)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8(wv[i], wv[i + 1], fw), widen8(xv[i], xv[i + 1], fx),
                                                          acc, 0, 0, 0);
        }
      }
    }
  }
  if (!live) return;
  with_act8(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const long n = n0 + 8 * (i / 4) + 4 * hi + i % 4;
      if (n >= a.n) continue;
      float v = acc[i] + a.bias[n];
      if (a.f32) {
        if (a.add) v += ((const float *)a.add)[r * a.as + n];
        ((float *)a.y)[r * a.ys + n] = act8<decltype(act)::value>(v);
      } else {
        if (a.add) v += (float)((const _Float16 *)a.add)[r * a.as + n];
        ((_Float16 *)a.y)[r * a.ys + n] = (_Float16)act8<decltype(act)::value>(v);
      }
    }
  });
}

}  // namespace
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
  a.act = act;
  a.add = d_add;
  a.as = (long)add_stride;
  IEN_CHECK((rows + 31) / 32 < 65536, IEN_ERR_INPUT, "%zu rows", rows);
  hipLaunchKernelGGL(k_multiply8, dim3((unsigned)(w->npad / 128), (unsigned)((rows + 31) / 32)), dim3(256), 0,
                     ctx->stream, a);
  IEN_HIP(hipGetLastError());
  return IEN_OK;
}

}  // extern "C"
