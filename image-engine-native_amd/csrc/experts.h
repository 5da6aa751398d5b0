// experts.h -- the plan of a routing (ien_routes) and the experts' weights
// (ien_experts8), shared by route.hip, experts_in8.hip and experts_out8.hip
// (internal).
#pragma once

#include "eight_bits.h"

// Weights in 8 bits, an expert's panels after another's: panel e cb + b (expert
// e, block b of 128 channels) as ien_matrix8's.  Gated, outputs lie in turns of
// 32: 32 gates, then the 32 they multiply; npad is then twice the outputs in
// whole 128s, else n in whole 128s.  SLACK8 more panels follow, of the tiles'
// loads ahead, and 128 rows.
struct ien_experts8 {
  ien_ctx *ctx = nullptr;
  size_t experts = 0, c = 0, n = 0;  // n: the outputs (of a gated product half the columns)
  int gated = 0, cb = 0;
  long npad = 0;
  uint8_t *d_w = nullptr;
  uint32_t *d_scales = nullptr;
  float *d_bias = nullptr;  // npad floats an expert, zero padded
};

namespace ien {

constexpr size_t MAX_EXPERTS = 1024, MAX_TOP = 16, MAX_PAIRS = (size_t)1 << 28;

// The rows of the tiles that a plan lists.
constexpr int TILE_SIZES = 4;
constexpr int TILE_ROWS[TILE_SIZES] = {16, 64, 128, 256};

// A tile: rows begin .. end of the order, of one expert.
struct ExpertTile {
  int expert, begin, end, unused;
};

// Where a plan's parts lie, in ints.
struct PlanLayout {
  long offsets, order, place;  // experts + 1; pairs; pairs (a pair's place in the order, -1 for none)
  long totals;                 // tiles of each size
  long tiles[TILE_SIZES];      // ExpertTile each
  long most[TILE_SIZES];       // of them, at most
  long parts, pitch;           // [chunk][pitch] counts of the chunks' pairs by expert, and without one
  long chunk, chunks;          // tokens
  long ints;
};

// Tokens are counted in chunks of 64s, at most 256 of them (every workgroup that
// places a chunk's pairs adds all chunks' counts).
inline PlanLayout plan_layout(size_t tokens, size_t experts, size_t top) {
  const long pairs = (long)(tokens * top), e = (long)experts;
  auto whole = [](long n) { return (n + 3) / 4 * 4; };
  PlanLayout p{};
  p.order = whole(e + 1);
  p.place = p.order + whole(pairs);
  p.totals = p.place + whole(pairs);
  long at = p.totals + TILE_SIZES;
  for (int s = 0; s < TILE_SIZES; s++) {
    p.tiles[s] = at;
    p.most[s] = pairs / TILE_ROWS[s] + std::min(pairs, e);
    at += 4 * p.most[s];
  }
  p.chunk = 64 * std::max(1L, ((long)tokens + 64 * 256 - 1) / (64 * 256));
  p.chunks = std::max(1L, ((long)tokens + p.chunk - 1) / p.chunk);
  p.parts = at;
  p.pitch = whole(e + 1);
  p.ints = at + p.chunks * p.pitch;
  return p;
}

// experts_in8.hip, experts_out8.hip: the tile of a product (gated 2: with the coarser sums).
int experts_in_choice(int cus, long pairs, long experts, long npad, int chunks, int gated);
int experts_out_choice(long pairs, long experts, int chunks);

// The routes that an entry point was handed, or its refusal.
ien_status check_routes(const ien_routes *r, const char *what);

}  // namespace ien
