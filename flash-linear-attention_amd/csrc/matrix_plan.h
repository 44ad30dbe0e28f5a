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

// Which tile and how many slices of the contraction, by an estimate of the time of each; from `most` on in size.  What it rests on (us for a slice of 128 bytes of k of
// every tile on a CU, measured in products of 70 to 8192 rows, bf16):
//                        256 x 256, one a CU       128 x 128, one and two   64 x 128, one, two and three
//   both contiguous      1.05 (few CUs) to 1.6     1.25  1.7                0.9   1.5   1.95
//   one or both strided  1.05 to 1.6               0.72  0.97               0.58  0.65  0.9
// Rows of 128 bytes out of two weights come slower than the strided operand's 256 and 512 bytes on end: where both are contiguous the tile with the fewest bytes wins early.
// Rows in 8-bit integers are decided by the same rates, which were not measured for them: a slice has the same bytes, and bytes are what bounds the smaller tiles.
// Ends: 12, 8 and 7 us for the first tile of a CU, half of that for each further one; sums of slices go out and in at 5 TB/s behind 5 us.
// Measured with all three tiles and 1 to 8 slices (us; M x K to F): forward 70 x 2048 to 5632: 28 - 47, taken 30; 200 x 4096 to 11008: 70 - 168, taken 70; 500 x 4096 to 4096: 65 - 140, taken 65;
// 1003 x 1000 to 2731: 35 - 95, taken 35.  dx of the last: 29 - 120, taken 29; of 2048 x 2048 to 5632: 100 - 208, taken 100; its weights' gradients 92 - 146, taken 92.
TilePlan plan_tiles(int64_t M, int64_t N, int64_t slices, int batch, bool contiguous, TileKind most = kBig) {
  constexpr double kEnds[3] = {12, 8, 7}, kSlice[2][3][3] = {{{0, 0, 0}, {0.72, 0.97, 0}, {0.58, 0.65, 0.9}}, {{0, 0, 0}, {1.25, 1.7, 0}, {0.9, 1.5, 1.95}}};
  TilePlan best{most, 1};
  double time = 0;
  for (int t = most; t < 3; ++t) {
    const int64_t tiles = batch * fla_cdiv(M, kTileM[t]) * fla_cdiv(N, kTileN[t]), room = kCUs * kTilePerCu[t];
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && (slices < 4 * splits || tiles * splits > 1024)) break;
      const int64_t n = tiles * splits, rounds = n / room, rest = n % room;
      auto slice = [&](int64_t on) { return t == kBig ? 1.05 + 0.55 * (double)on / kCUs : kSlice[contiguous][t][fla_cdiv(on, kCUs) - 1]; };
      double last = rest ? slice(rest) : 0;
      if (t == kBig && splits == 1 && rest_in_halves(n)) last = 0.6 * slice(kCUs);
      const int64_t turns = rounds + (rest > 0);
      double est = (double)fla_cdiv(slices, splits) * ((double)rounds * slice(room) + last) + kEnds[t] * (0.5 + 0.5 * (double)turns);
      if (splits > 1) est += 5 + 8 * splits * batch * (double)M * (double)N / 5e6;
      if ((t == most && splits == 1) || est < time) best = {(TileKind)t, splits}, time = est;
    }
  }
  best.splits = (int)fla_cdiv(slices, fla_cdiv(slices, best.splits));   // none of them empty
  return best;
}

// ... of the products there are.  Up to kPanelRows rows of x those of contiguous operands go to the panels instead.
constexpr int64_t kPanelRows = 64;
TilePlan plan_gated(int64_t M, int64_t F, int64_t row_bytes) { return plan_tiles(M, 2 * F, fla_cdiv(row_bytes, kSliceBytes), 1, true); }
TilePlan plan_dx(int64_t M, int64_t F, int64_t K) { return plan_tiles(M, K, 2 * fla_cdiv(F * 2, kSliceBytes), 1, false); }
TilePlan plan_dw(int64_t M, int64_t F, int64_t K, int batch) { return plan_tiles(F, K, fla_cdiv(M, 64), batch, false); }
// (fp32 results leave in 128 x 128 tiles: the big one is built for 16 bits)
TilePlan plan_int8(int64_t M, int64_t N, int64_t K, bool big) { return plan_tiles(M, N, fla_cdiv(K, kSliceBytes), 1, true, big ? kBig : kMiddle); }

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
