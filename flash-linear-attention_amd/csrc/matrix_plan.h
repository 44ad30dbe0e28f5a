// Which tile of matrix_tiles.h a product takes, and how many slices its contraction is cut into.
#pragma once
#include <initializer_list>

#include "matrix_tiles.h"

namespace {

enum TileKind { kBig, kMiddle, kSmall };
struct TilePlan {
  TileKind kind;
  int splits;
};
constexpr int kCUs = 256;
constexpr int kTileM[3] = {256, 128, 64}, kTileN[3] = {256, 128, 128}, kTilePerCu[3] = {1, 2, 3};
// What is left behind whole rounds of big tiles goes in tiles of half the columns where a CU then has one at most
constexpr bool rest_in_halves(int64_t tiles) { return tiles % kCUs != 0 && tiles % kCUs <= kCUs / 2 && tiles > kCUs; }

// Which tile and how many slices of the contraction, by an estimate of the time of each.
// From `most` on in size.
TilePlan plan_tiles(int64_t M, int64_t N, int64_t slices, int batch, TileKind most = kBig) {
  // us for a slice of 128 bytes of k of a tile, with as many tiles on the CU as it holds, and for a half tile
  constexpr double kSlice[3] = {1.6, 0.49, 0.3}, kHalf = 0.6;
  TilePlan best{most, 1};
  double time = 0;
  for (int t = most; t < 3; ++t) {
    const int64_t tiles = batch * fla_cdiv(M, kTileM[t]) * fla_cdiv(N, kTileN[t]), room = kCUs * kTilePerCu[t];
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (slices < 4 * splits || tiles * splits > 1024)) break;
      const int64_t n = tiles * splits, rounds = fla_cdiv(n, room), in_last = n - (rounds - 1) * room;
      // a CU with some of its tiles missing runs the others faster, but not as much
      double last = 0.5 + 0.5 * (double)fla_cdiv(in_last, kCUs) / kTilePerCu[t];
      if (t == kBig && splits == 1 && rest_in_halves(n)) last = kHalf;
      double est = (double)(fla_cdiv(slices, splits) + 4) * kSlice[t] * kTilePerCu[t] * ((double)(rounds - 1) + last) + 3;
      if (splits > 1) est += 4 + 8 * splits * batch * (double)M * (double)N / 4e6;     // the sums go out and in
      if ((t == most && splits == 1) || est < time) best = {(TileKind)t, splits}, time = est;
    }
  }
  best.splits = (int)fla_cdiv(slices, fla_cdiv(slices, best.splits));   // none of them empty
  return best;
}

// The launch of tm rows of tn tiles
int grid_of(TileKind kind, int64_t tm, int64_t tn, int splits, MatGrid* g, dim3* grid) {
  const int64_t tiles = tm * tn;
  FLA_REQUIRE(tiles < (int64_t)1 << 24, FLA_E_UNSUPPORTED);   // (a launch is less than 2^32 threads)
  const bool turns = kind == kBig && splits == 1, halves = turns && rest_in_halves(tiles);
  const int64_t whole = halves ? tiles / kCUs * kCUs : tiles;
  *g = MatGrid{(uint32_t)tm, (uint32_t)tn, (uint32_t)whole, (uint32_t)(halves ? 2 * (tiles - whole) : 0)};
  *grid = dim3((unsigned)(turns && tiles > kCUs ? kCUs : tiles), splits);
  return FLA_OK;
}

bool sizes_ok(int64_t M, int64_t F, int64_t K) { return M <= 0x7fffffff && F <= kMatMaxDim && K <= kMatMaxDim; }
bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t any = 0;
  for (const void* p : ps) any |= (uintptr_t)p;
  return any % 16 == 0;
}

bool aligned4(std::initializer_list<const void*> ps) {
  uintptr_t any = 0;
  for (const void* p : ps) any |= (uintptr_t)p;
  return any % 4 == 0;
}

}  // namespace
