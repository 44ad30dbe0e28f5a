// Diagnostics: the tiles that a product is launched in.
#include "matrix_plan.h"

extern "C" int fla_selftest_matrix_plan(int product, int64_t M, int64_t N, int64_t K, int* plan) {
  FLA_REQUIRE(plan && product >= FLA_PRODUCT_GATED && product <= FLA_PRODUCT_INT8_F32 && M > 0 && N > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(sizes_ok(M, N, K), FLA_E_UNSUPPORTED);
  const bool dw = product == FLA_PRODUCT_GATED_DW || product == FLA_PRODUCT_GATED_DW1;
  for (int i = 0; i < 5; ++i) plan[i] = 0;
  if (M <= kPanelRows && product != FLA_PRODUCT_GATED_DX && !dw) return FLA_OK;
  const int batch = product == FLA_PRODUCT_GATED_DW ? 2 : 1;
  TilePlan t{};
  switch (product) {
    case FLA_PRODUCT_GATED: t = plan_gated(M, N, K * 2); break;
    case FLA_PRODUCT_GATED_INT8: t = plan_gated(M, N, K); break;
    case FLA_PRODUCT_GATED_DX: t = plan_dx(M, N, K); break;
    case FLA_PRODUCT_GATED_DW:
    case FLA_PRODUCT_GATED_DW1: t = plan_dw(M, N, K, batch); break;
    default: t = plan_int8(M, N, K, product == FLA_PRODUCT_INT8);
  }
  // rows and columns of the results, and columns of a tile (of h: half of the tile's, which holds both products)
  const bool gated = product == FLA_PRODUCT_GATED || product == FLA_PRODUCT_GATED_INT8;
  const int64_t rows = dw ? N : M, columns = product == FLA_PRODUCT_GATED_DX || dw ? K : N;
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(t.kind, batch * fla_cdiv(rows, kTileM[t.kind]), fla_cdiv(columns, kTileN[t.kind] / (gated ? 2 : 1)), t.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  plan[0] = kTileM[t.kind], plan[1] = t.splits, plan[2] = (int)grid.x, plan[3] = (int)g.whole, plan[4] = (int)g.halves;
  return FLA_OK;
}
