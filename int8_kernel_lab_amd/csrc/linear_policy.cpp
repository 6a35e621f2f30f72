// Which kernel runs an int8 linear layer: the policy of the linear layers, kept
// outside the kernels like that of the convolutions (policy.cpp).
#include <algorithm>
#include <cmath>

#include "i8conv_internal.hpp"
#include "linear_common.hpp"

namespace i8conv {
namespace {

// A tile of kernel_linear.hip and what it takes, in us: a 128-byte k-stage with
// one workgroup on a compute unit and few of them busy (`alone`), with all of
// them full (`full`), and what a tile costs besides its stages.  Read off
// sweeps of 80 to 4096 rows over 1024 to 12288 columns, 1024 to 8192 deep, on
// all tiles.
struct TileCost {
  int tile, bm, bn, per_unit, kg, buffers;
  bool plain, gated;
  double alone, full, besides;
};
const TileCost kTiles[] = {
    {kTile256x256, 256, 256, 1, 1, 2, true, true, 1.25, 1.80, 10.0},
    {kTile128x256, 128, 256, 1, 1, 3, true, true, 0.76, 1.10, 6.0},
    {kTile128x128, 128, 128, 2, 1, 2, true, true, 0.66, 1.18, 5.0},
    {kTile128x64, 128, 64, 3, 1, 2, true, true, 0.60, 1.05, 3.5},
    {kTile64x64, 64, 64, 4, 1, 2, true, false, 0.50, 0.90, 2.5},
    {kTile64x64Deep, 64, 64, 2, 1, 4, true, false, 0.28, 0.45, 2.5},
    {kTile64x64Pair, 64, 64, 1, 2, 4, true, false, 0.42, 0.50, 2.5},
    {kTile128x64Pair, 128, 64, 1, 2, 3, false, true, 0.60, 0.76, 3.0},
};

// Row tiles as rounds of the chip, the last of them as full as it is.  (A part of
// a tile counts as a whole one: at 0.8 of it the choice for 300 drawn layers by
// expert lay 3.7 % from the best tile in the mean, so 1.6 %.)
double cost(const TileCost &t, double row_tiles, int64_t wide, int64_t k) {
  const double tiles = row_tiles * double((wide + t.bn - 1) / t.bn);
  const double slots = 256.0 * t.per_unit, rounds = std::floor(tiles / slots);
  const double fill = tiles / slots - rounds;
  const double stages = double((k + 128 * t.kg - 1) / (128 * t.kg));
  double us = rounds * (stages * t.full + t.besides);
  if (fill > 0) us += stages * (t.alone + (t.full - t.alone) * fill) + t.besides;
  return us;
}

}  // namespace

const char *linear_tile_name(int tile) {
  switch (tile) {
    case kTile256x256: return "256 rows x 256";
    case kTile128x256: return "128 rows x 256";
    case kTile128x128: return "128 rows x 128";
    case kTile128x64: return "128 rows x 64";
    case kTile128x64Pair: return "128 rows x 64, two groups of waves";
    case kTile64x64: return "64 rows x 64";
    case kTile64x64Deep: return "64 rows x 64, four stages";
    case kTile64x64Pair: return "64 rows x 64, two groups of waves";
  }
  return "?";
}

int plan_linear_tile(int64_t rows, int64_t experts, int64_t n, int64_t k, bool gated) {
  int best = kTile128x128;
  double least = 1e300;
  for (const TileCost &t : kTiles) {
    if (gated ? !t.gated : !t.plain) continue;
    // the LDS of every workgroup of a unit (launch_tile has the same sum)
    const int64_t lds = int64_t(t.kg) * t.buffers * (t.bm + t.bn) * kStageBytes +
                        8 * (2 * t.bn + t.bm) + (experts ? 8 * (experts + 1) : 0);
    if (lds * t.per_unit > kLdsBudget) continue;
    double row_tiles = double((rows + t.bm - 1) / t.bm);
    if (experts) {
      // each group ends in a part of a tile, in the mean half of one
      const double groups = double(std::min(experts, rows));
      row_tiles = std::max(0.0, double(rows) / t.bm - groups / 2) + groups;
    }
    const double us = cost(t, row_tiles, gated ? 2 * n : n, k);
    if (us < least) least = us, best = t.tile;
  }
  return best;
}

}  // namespace i8conv
