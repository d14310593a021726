// Tiles of the dense products on CTA pairs (mmoe_dense.cu): their sizes, and how many columns those of a launch have.  Host code only.
#pragma once

#include <algorithm>

#include "mmoe_dense.cuh"

namespace mmoe {

constexpr int kPairRows = 128;                        // rows of A per CTA
constexpr int kPairCols = 256;                        // most rows of B per tile
constexpr int kStageA = kPairRows * 128;              // bytes
constexpr int kMaxStages = 9;                         // what fits of the narrowest tiles, 64 columns
constexpr int kEpiWarps = 8;                          // two per TMEM lane quadrant, each with every other block of columns
constexpr int kEpiBlock = 32 * 32 * 4;                // a warp's 32 rows x 32 sums on their way from lanes to rows
constexpr int kPairThreads = 32 * (2 + kEpiWarps);
constexpr int kPairSmem = 227 * 1024;
constexpr int kPairStageRoom = kPairSmem - 1024 - 1024 - kEpiWarps * kEpiBlock;
static_assert(kPairStageRoom / (kStageA + 32 * 128) == kMaxStages, "stages of the narrowest tiles");

// bytes of B that a stage of a tile holds in each CTA
inline int stage_b_bytes(const DenseProduct& p, int cols) { return p.b.k_rows ? (cols / 2 + 63) / 64 * 8192 : cols / 2 * 128; }

// What a tile of a product costs on a pair, in clocks: a stage 2.1 a column in the tensor cores, or its bytes at 60 a clock into each SM; the
// epilogue 24 a column, beside the next tile's products or, of the last tile, behind them.
struct TileCost {
  int64_t tiles, products, epilogue;
};
inline TileCost tile_cost(const DenseProduct& p, int cols) {
  const int width = p.kind == kGated ? cols / 2 : cols, depth = p.type == kDenseInt8 ? 128 : 64;
  const int64_t m_tiles = (p.m + 2 * kPairRows - 1) / (2 * kPairRows);
  return TileCost{m_tiles * ((p.n + width - 1) / width),
                  (int64_t)((p.k + depth - 1) / depth) * std::max((kStageA + stage_b_bytes(p, cols)) / 60, 21 * cols / 10), 24 * cols};
}

// Columns of each product's tiles: those with which the pair that has most to do ends first.  Against 256 columns always: 8-bit projection of 777
// tokens, 5120 x 5120, 33.4 -> 23.8 us (160 columns, two turns of 128 tiles where 256 have two of 80), 16-bit block of 1021 tokens 60.5 ->
// 57.5, 8-bit gated product of 256 tokens 17.2 -> 11.9 (64 columns); 3840 tokens the same within 1 %.
inline void choose_cols(const DenseProduct* p, int parts, int pairs, int (&best)[kMaxParts]) {
  constexpr int kChoices = kPairCols / 32 - 1;          // 256, 224 ... 64
  TileCost cost[kMaxParts][kChoices] = {};
  for (int i = 0; i < parts; ++i)
    for (int c = 0; c < kChoices; ++c) cost[i][c] = tile_cost(p[i], kPairCols - 32 * c);
  int64_t least = INT64_MAX;
  for (int c0 = 0; c0 < kChoices; ++c0)
    for (int c1 = 0; c1 < (parts > 1 ? kChoices : 1); ++c1) {
      const TileCost &x = cost[0][c0], &y = cost[1][c1];
      // the pairs with most tiles of the first, and those with one less
      const int64_t all = (x.tiles + y.tiles + pairs - 1) / pairs, most = (x.tiles + pairs - 1) / pairs;
      int64_t longest = 0;
      for (int64_t first = x.tiles / pairs; first <= most; ++first) {
        const int64_t second = std::max<int64_t>(0, all - first);
        longest = std::max(longest, first * std::max(x.products, x.epilogue) + second * std::max(y.products, y.epilogue) + (second > 0 ? y.epilogue : x.epilogue));
      }
      if (longest < least) least = longest, best[0] = kPairCols - 32 * c0, best[1] = kPairCols - 32 * c1;
    }
}

}  // namespace mmoe
