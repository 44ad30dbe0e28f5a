// Products of rows in 8-bit integers with results in bf16, and the library's entries.
#include "int8_linear.h"

// int8_linear_f16.hip, int8_linear_f32.hip (p: an Int8Params)
int fla_int8_linear_f16(void* p, hipStream_t st);
int fla_int8_linear_f32(void* p, hipStream_t st);

extern "C" int fla_int8_linear_splits(int64_t M, int64_t N, int64_t K, int dtype) {
  return M <= kPanelRows || N <= 0 || K <= 0 ? 1 : plan_int8(M, N, K, dtype != FLA_F32).splits;
}

extern "C" int fla_int8_linear(const void* x, const float* x_scale, const void* weight, const float* weight_scale, const void* bias,
                               int bias_dtype, const void* residual, int residual_dtype, void* y, int64_t M, int64_t N, int64_t K,
                               int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && weight && weight_scale && y && M >= 0 && N > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16 || dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!bias || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual || residual_dtype == dtype || residual_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, N, K) && K % 16 == 0 && K <= FLA_INT8_MAX_K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, weight, workspace}) && aligned4({bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  Int8Params p{};
  p.x = (const char*)x, p.w = (const char*)weight, p.sx = x_scale, p.sw = weight_scale, p.bias = bias, p.res = residual, p.y = y;
  p.part = (int*)workspace, p.M = M, p.N = N, p.K = K, p.act = activation, p.splits = 1;
  p.bias_f32 = bias_dtype == FLA_F32, p.res_f32 = residual_dtype == FLA_F32;
  p.res_wide = N % 4 == 0 && (uintptr_t)residual % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_int8<bf16>(p, st) : dtype == FLA_F16 ? fla_int8_linear_f16(&p, st) : fla_int8_linear_f32(&p, st);
}
