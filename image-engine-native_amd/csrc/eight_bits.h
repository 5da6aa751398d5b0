// eight_bits.h -- rows in 8 bits (ien_rows8) and weights in 8 bits, shared by
// quantize8.hip, multiply8.hip and group_norm.hip (internal).
#pragma once

#include "conv_common.h"
#include "lanes.h"

// Weights in 8 bits: panel t cb + b (tap t, block b of 128 channels) holds
// npad rows of 128 e4m3 bytes, an output each (zeros past c and n), and npad
// scale dwords (the byte in the low 8 bits); npad is n in whole 128s.  A
// tile's share of a panel is one contiguous piece.  SLACK8 more panels and 128
// rows and scales follow (not set: no stored output comes from them): tiles of
// 256 outputs and the loads ahead of the last block read that far.
struct ien_matrix8 {
  ien_ctx *ctx = nullptr;
  size_t taps = 0, c = 0, n = 0;
  int cb = 0;
  long npad = 0;
  uint8_t *d_w = nullptr;
  uint32_t *d_scales = nullptr;
  float *d_bias = nullptr;  // npad floats, zero padded
};

namespace ien {

constexpr int BLOCK8 = 128;  // values under one scale
constexpr int SLACK8 = 4;    // panels of weights past the last one

inline size_t blocks8(size_t k) { return (k + BLOCK8 - 1) / BLOCK8; }

// Rows in 8 bits that an entry point was handed, or its refusal.
ien_status check_rows8(const ien_rows8 *r, size_t k, const char *what);

// quantize8.hip: workgroups for rows of that many blocks in all.
unsigned quantize8_grid(long blocks);

// group_norm.hip: the launches of a norm of `images` maps of `pixels` pixels, c
// channels in `groups` groups, into results of y_bytes.
struct NormPlan {
  long one;     // one launch (or two, over `chunks` parts of an image of `chunk` pixels)
  long span;    // channels a workgroup handles (c, or a part in one launch)
  long px;      // pixels side by side in one launch
  long chunks, chunk;
  long lanes;   // of a workgroup
  long groups;  // workgroups an image
  long images;  // of a turn: no launch has 2^32 lanes, and their parts fit the workspace
};
NormPlan norm_plan(int cus, long workspace, long images, long pixels, int c, int groups, int y_bytes);

// multiply8.hip: 64 x the tile + the splits of the depth of a product of `rows`
// rows, `chunks` blocks deep, n outputs.
int multiply8_choice(int cus, long workspace, long rows, long n, int chunks, bool exact, bool add);
// The rows of one launch of that tile, at most.
long multiply8_part(int tile, long n);

typedef int int2v __attribute__((ext_vector_type(2)));

// The exponent of a block whose largest finite magnitude is `largest`: the
// smallest e >= -127 with largest <= 448 2^e = 1.75 2^(e + 8), 0 for zero.
__device__ __forceinline__ int exponent8(float largest) {
  const uint32_t b = __float_as_uint(largest);
  const int e = (int)(b >> 23) - 135 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
  return b == 0 ? 0 : e < -127 ? -127 : e;
}

// 2^-e for the e that exponent8 gives (-127 .. 120): a normal f32.
__device__ __forceinline__ float inverse_power(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }

// 2^(scale - 127) for scales 0 .. 254.
__device__ __forceinline__ float scale_power(int scale) {
  return __uint_as_float(scale == 0 ? 0x00400000u : (uint32_t)scale << 23);
}

__device__ __forceinline__ bool finite8(float v) { return (__float_as_uint(v) & 0x7f800000) != 0x7f800000; }
__device__ __forceinline__ float finite_magnitude(float v) { return finite8(v) ? fabsf(v) : 0.0f; }

// Eight values times the power of two `inv` as e4m3 bytes, to nearest even
// (finite ones are within 448 by the block's scale; others become NaN).
__device__ __forceinline__ int2v pack8(const float *v, float inv) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; i++) s[i] = finite8(v[i]) ? v[i] * inv : __uint_as_float(0x7fc00000);
  int2v r;
  r.x = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  r.x = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], r.x, true);
  r.y = __builtin_amdgcn_cvt_pk_fp8_f32(s[4], s[5], 0, false);
  r.y = __builtin_amdgcn_cvt_pk_fp8_f32(s[6], s[7], r.y, true);
  return r;
}

// The largest of v over each aligned group of 16 lanes, in all of them.
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_from<0xB1>(v));
  v = fmaxf(v, dpp_from<0x4E>(v));
  v = fmaxf(v, dpp_from<0x141>(v));
  return fmaxf(v, dpp_from<0x140>(v));
}

typedef half8 half8_any __attribute__((aligned(2)));
typedef float4v float4_any __attribute__((aligned(4)));

// Eight consecutive values from channel `at` of a row of c (T: f16 or f32),
// zeros past c; VEC: the whole eight in 16-byte loads, at any element.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *row, long at, long c, float *v) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 2) {
      const half8 h = *(const half8_any *)(row + at);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = (float)h[i];
    } else {
      const float4v a = *(const float4_any *)(row + at), b = *(const float4_any *)(row + at + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = at + i < c ? (float)row[at + i] : 0.0f;
  }
}

// Their counterpart: f16 rounds to nearest even.
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *row, long at, long c, const float *v) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 2) {
      half8 h;
#pragma unroll
      for (int i = 0; i < 8; i++) h[i] = (_Float16)v[i];
      *(half8_any *)(row + at) = h;
    } else {
      *(float4_any *)(row + at) = float4v{v[0], v[1], v[2], v[3]};
      *(float4_any *)(row + at + 4) = float4v{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (at + i < c) row[at + i] = (T)v[i];
  }
}

// Eight results of a row.  In f16 past the caches' order of use, for what no
// cache would hold until it is read (it would put out what is still to be read:
// 16384 rows 2048 -> 8192 with fast sums 295 -> 248 us, the norm of 512 x 768 x 128 64 -> 54).
// f32 results go in two halves of a line a wave, which the caches have to join
// (without them 98304 rows of 512 98 -> 115 us).
template <typename T>
__device__ __forceinline__ void stream8(T *at, const float *v) {
  if constexpr (sizeof(T) == 2) {
    half8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (_Float16)v[i];
    __builtin_nontemporal_store(h, (half8_any *)at);
  } else {
    store8<T, true>(at, 0, 0, v);
  }
}

inline bool act8_known(ien_act act) {
  return act == IEN_ACT_NONE || act == IEN_ACT_RELU || act == IEN_ACT_GELU || act == IEN_ACT_SIGMOID ||
         act == IEN_ACT_SILU;
}

// GELU for f32 results: v Phi(v) = max(v, 0) - a Phi(-a), a = |v|, with
// Phi(-a) = e^(-a^2/2) Q(t), Q a polynomial of t = 1 / (1 + 0.3 a) fitted here by
// least squares for a up to 15 (6e-8 of Phi), past which it is 0.  The tail is off
// by some steps of f32 and by v^2 steps where it is small; the result at most by
// 1.4e-7 in -3 .. 3 and 3e-9 in -6 .. -3 (v (1 + erf(v / sqrt 2)) / 2 in f32: 2.5e-7
// and 8e-8), and -0 at -infinity; gelu_f, made for results in f16, is off by 5.6e-7,
// 1.3e-6 and, below -6, 3e-8 of v.  An exponential dearer than gelu_f: 4096 rows
// 384 -> 1536 11.3 -> 12.1 us.
__device__ __forceinline__ float gelu8(float v) {
  const float a = fminf(fabsf(v), 15.0f), t = __builtin_amdgcn_rcpf(1.0f + 0.3f * a);
  float q = 0.03842524066567421f;
  q = q * t - 0.16939404606819153f;
  q = q * t + 0.22913022339344025f;
  q = q * t - 0.07704316824674606f;
  q = q * t + 0.1429053395986557f;
  q = q * t + 0.09452646225690842f;
  q = q * t + 0.12196037918329239f;
  q = q * t + 0.11948210000991821f;
  q = q * t + 7.494882538594538e-06f;
  const float e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);  // (log2(e) / 2)
  return (v < 0.0f ? 0.0f : v) - a * (q * e);  // (a NaN stays one)
}

template <int ACT>
__device__ __forceinline__ float act8(float v) {
  if constexpr (ACT == IEN_ACT_GELU) return gelu8(v);
  else if constexpr (ACT == IEN_ACT_SILU)
    return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v));  // (1 ulp; past e^88 the result is -0)
  else if constexpr (ACT == IEN_ACT_RELU) return v < 0.0f ? 0.0f : v;  // (a NaN stays one)
  else return act_c<ACT>(v, 0.0f);
}

// f(Act<...>) with the activation as a compile-time choice.
template <int A>
struct Act {
  static constexpr int value = A;
};
template <typename F>
__device__ __forceinline__ void with_act8(int act, F f) {
  switch (act) {
    case IEN_ACT_RELU: f(Act<IEN_ACT_RELU>{}); break;
    case IEN_ACT_GELU: f(Act<IEN_ACT_GELU>{}); break;
    case IEN_ACT_SIGMOID: f(Act<IEN_ACT_SIGMOID>{}); break;
    case IEN_ACT_SILU: f(Act<IEN_ACT_SILU>{}); break;
    default: f(Act<IEN_ACT_NONE>{}); break;
  }
}

}  // namespace ien
