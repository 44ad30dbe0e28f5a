// Which tile of matrix_tiles.h a product takes, and how many slices its contraction is cut into.
#pragma once
#include <initializer_list>

#include "matrix_tiles.h"

namespace {

// Which tile and how many slices of the contraction: the estimated time of each, in slices' time of a CU.
enum TileKind { kBig, kMiddle, kSmall };
struct TilePlan {
  TileKind kind;
  int splits;
};
constexpr int kTileM[3] = {256, 128, 64}, kTileN[3] = {256, 128, 128}, kTilePerCu[3] = {1, 2, 3};
TilePlan plan_tiles(int64_t M, int64_t N, int64_t slices, int batch, double bytes_per_sum) {
  // us for a slice of 128 bytes of k of a tile, with as many tiles on the CU as it holds
  constexpr double kSlice[3] = {1.55, 0.55, 0.36};
  TilePlan best{kBig, 1};
  double time = 0;
  for (int t = 0; t < 3; ++t) {
    const int64_t tiles = batch * fla_cdiv(M, kTileM[t]) * fla_cdiv(N, kTileN[t]);
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (slices < 4 * splits || tiles * splits > 1024)) break;
      const int64_t n = tiles * splits, rounds = fla_cdiv(n, 256 * kTilePerCu[t]), in_last = n - (rounds - 1) * 256 * kTilePerCu[t];
      // a CU with some of its tiles missing runs the others faster, but not as much
      const double last = 0.5 + 0.5 * (double)fla_cdiv(in_last, 256) / kTilePerCu[t];
      double est = (double)(fla_cdiv(slices, splits) + 4) * kSlice[t] * kTilePerCu[t] * ((double)(rounds - 1) + last) + 3;
      if (splits > 1) est += 4 + 2 * splits * bytes_per_sum * batch * (double)M * (double)N / 4e6;
      if ((t == 0 && splits == 1) || est < time) best = {(TileKind)t, splits}, time = est;
    }
  }
  best.splits = (int)fla_cdiv(slices, fla_cdiv(slices, best.splits));   // none of them empty
  return best;
}

constexpr int64_t kMaxGrid = (int64_t)1 << 24;   // workgroups of 256 threads in a launch of less than 2^32

bool sizes_ok(int64_t M, int64_t F, int64_t K) { return M <= 0x7fffffff && F <= kMatMaxDim && K <= kMatMaxDim; }
bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t any = 0;
  for (const void* p : ps) any |= (uintptr_t)p;
  return any % 16 == 0;
}

}  // namespace
