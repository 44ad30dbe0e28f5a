// The gated product of rows in 8-bit integers.
#include "gated_forward.h"

extern "C" int fla_int8_gated_linear_fwd(const void* x, const float* x_scale, const void* gate_weight, const float* gate_scale, const void* up_weight,
                                         const float* up_scale, const void* gate_bias, const void* up_bias, int bias_dtype, void* h, int64_t M,
                                         int64_t F, int64_t K, int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && gate_weight && gate_scale && up_weight && up_scale && h && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!gate_bias && !up_bias) || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 16 == 0 && K <= FLA_INT8_MAX_K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, gate_weight, up_weight, workspace}) && aligned4({gate_bias, up_bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedParams p{};
  p.x = (const char*)x, p.wg = (const char*)gate_weight, p.wu = (const char*)up_weight, p.sx = x_scale, p.sg = gate_scale, p.su = up_scale;
  p.bg = gate_bias, p.bu = up_bias, p.h = h, p.part = workspace, p.M = M, p.F = F, p.K = K, p.ldk = (F + 7) / 8 * 8;
  p.act = activation, p.bias_f32 = bias_dtype == FLA_F32;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? gated_forward<int8_t, bf16>(p, st) : gated_forward<int8_t, f16>(p, st);
}
