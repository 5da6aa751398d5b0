// few8.h -- the experts' products where an expert has few rows (internal): a
// workgroup takes up to 16 of them and reads its share of the weights once,
// straight from memory into the registers of v_mfma_f32_16x16x32_bf16.
//
// Memory bounds it, so nothing is staged: a lane's two 16 bytes of a block of 128 are
// four products' operands (the order of a sum's terms is any, as long as rows and
// weights have the same), four blocks are under way at a time (eight: the same), and
// the weights' addresses wait for the tile's expert alone, not for its rows.  Products
// are those of ien_multiply8's default (bf16 operands, sums in f32), whatever the
// caller asks for: the matrix pipe has nothing else to do.  32 tokens, four of 64 experts
// each, 1024 -> 2 x 1024 gated: 24.1 us, 4.8 TB/s of the weights of the 56 experts that
// have a token; 15.3 us where the tokens share 10 to 14 of them.
#pragma once

#include "tile8.h"

namespace ien {
namespace {

// WN x WK waves: 16 outputs each (gated: and the 16 they multiply), a WK-th of the
// depth.  Into rows in 8 bits WN is 8, a block of 128 outputs.
template <Kind8 KIND, typename Y, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) void k_few8(Args8 a) {
  constexpr int TILES = KIND == EXPERTS_GATED8 ? 2 : 1, AHEAD = 4, ROWS = TILE_ROWS[0];
  static_assert(KIND == EXPERTS_ROWS8 || WN == 8, "a block of outputs");
  __shared__ float4v sums[WK > 1 ? (WK - 1) * WN * TILES * 64 : 1];
  __shared__ float maxima[WN][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, part = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wk = wave / WN;
  const int tile = blockIdx.x / a.tiles_n;
  const long o0 = (long)(blockIdx.x - tile * a.tiles_n) * WN * 16 + wn * 16;  // this wave's first output
  const ExpertTile t = a.list[tile];  // (past the last: whatever was there)
  if (tile >= *a.total) return;
  const long expert = t.expert;
  const int rows = t.end - t.begin;

  // This lane's columns: of output o0 + r, and gated its factor's, 32 further on.
  const long column = KIND == EXPERTS_GATED8 ? o0 / 32 * 64 + o0 % 32 + r : o0 + r;
  const bool outs = column + 32 * (TILES - 1) < a.npad;  // (the same for the wave: npad is whole 128s)
  const uint8_t *w = a.w + (expert * a.cb * a.npad + (outs ? column : 0)) * BLOCK8 + 16 * part;
  const uint32_t *ws = a.ws + expert * a.cb * a.npad + (outs ? column : 0);
  const int each = (a.cb + WK - 1) / WK, from = wk * each, to = min(from + each, a.cb);
  long row = t.begin + min(r, rows - 1);
  if constexpr (KIND >= EXPERTS_ACT8) row = a.order[row] / a.top;
  const uint8_t *x = a.x + row * a.xs + 16 * part, *xscale = a.scales + row * a.ss;

  float4v acc[TILES] = {};
  for (int b0 = from; b0 < to; b0 += AHEAD) {
    int4v wv[AHEAD][TILES][2], xv[AHEAD][2];
    int wsv[AHEAD][TILES], xsv[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      const long b = min(b0 + k, to - 1);
#pragma unroll
      for (int j = 0; j < TILES; j++) {
        const int4v *p = (const int4v *)(w + (b * a.npad + 32 * j) * BLOCK8);
        wv[k][j][0] = p[0], wv[k][j][1] = p[4];
        wsv[k][j] = (int)ws[b * a.npad + 32 * j];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      const long b = min(b0 + k, to - 1);
      const int4v *p = (const int4v *)(x + b * BLOCK8);
      xv[k][0] = p[0], xv[k][1] = p[4];
      xsv[k] = xscale[b];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      const bool on = r < rows && b0 + k < to;
      const float xp = scale_power(xsv[k]);
#pragma unroll
      for (int j = 0; j < TILES; j++) {
        const float wp = scale_power(wsv[k][j]);
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const int lo = s / 2, at = 2 * (s % 2);
          const bf16x8 xb = widen8(on ? xv[k][lo][at] : 0, on ? xv[k][lo][at + 1] : 0, xp);
          const bf16x8 wb = widen8(wv[k][j][lo][at], wv[k][j][lo][at + 1], wp);
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, xb, acc[j], 0, 0, 0);
        }
      }
    }
  }
  if constexpr (WK > 1) {
#pragma unroll
    for (int j = 0; j < TILES; j++)
      if (wk > 0) sums[(((wk - 1) * WN + wn) * TILES + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int k = 0; k < WK - 1; k++)
#pragma unroll
        for (int j = 0; j < TILES; j++) acc[j] += sums[((k * WN + wn) * TILES + j) * 64 + lane];
    }
  }

  // A lane has outputs o0 + 4 part .. + 3 of row r.
  const long at = o0 + 4 * part;
  const float *bias = a.bias + expert * a.npad + (outs ? column - r + 4 * part : 0);
  if constexpr (KIND == EXPERTS_ROWS8) {
    if (wk > 0 || r >= rows || at >= a.ys) return;  // (rows of parts are whole eights)
    const float4v v = acc[0] + *(const float4v *)bias;
    Y *y = (Y *)a.y + (t.begin + r) * a.ys + at;
    if constexpr (sizeof(Y) == 2) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4)));
      *(half4 *)y = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
      *(float4v *)y = v;
    }
  } else {
    float v[4], m = 0.0f;
    with_act8(a.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[e] = act8<decltype(act)::value>(acc[0][e] + bias[e]);
        if constexpr (KIND == EXPERTS_GATED8) v[e] *= acc[TILES - 1][e] + bias[32 + e];
        if (at + e >= a.n) v[e] = 0.0f;
        m = fmaxf(m, finite_magnitude(v[e]));
      }
    });
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    if (wk == 0 && part == 0) maxima[wn][r] = m;
    __syncthreads();
    if (wk > 0 || r >= rows) return;
#pragma unroll
    for (int k = 0; k < WN; k++) m = fmaxf(m, maxima[k][r]);
    const int e = exponent8(m);
    const float pad[8] = {v[0], v[1], v[2], v[3]};
    *(int *)(a.q + (t.begin + r) * a.qstride + at) = pack8(pad, inverse_power(e)).x;
    if (part == 0 && wn == 0) a.qs[(t.begin + r) * a.qsstride + at / BLOCK8] = (uint8_t)(e + 127);
  }
}

// A launch counts its lanes in 32 bits.
inline bool launches(long tiles_m, int tiles_n, int threads) { return tiles_m * tiles_n < (1L << 32) / threads; }

template <Kind8 KIND, typename Y, int WN, int WK>
bool launch_few(ien_ctx *ctx, Args8 &a, const ien_routes *r, const PlanLayout &p) {
  a.tiles_n = (int)((a.n + 16 * WN - 1) / (16 * WN));
  a.list = (const ExpertTile *)(r->d_plan + p.tiles[0]);
  a.total = r->d_plan + p.totals;
  if (!launches(p.most[0], a.tiles_n, 64 * WN * WK)) return false;
  hipLaunchKernelGGL((k_few8<KIND, Y, WN, WK>), dim3((unsigned)(p.most[0] * a.tiles_n)), dim3(64 * WN * WK), 0,
                     ctx->stream, a);
  return true;
}

}  // namespace
}  // namespace ien
