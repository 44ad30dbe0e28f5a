// The gated product of bf16 rows, and the library's entries for 16-bit rows.
#include "gated_forward.h"

int fla_gated_linear_f16(void* p, hipStream_t st);   // gated_f16.hip (p: a GatedParams)

extern "C" int fla_gated_linear_splits(int64_t M, int64_t F, int64_t K, int element_bytes) {
  return M <= kPanelRows || F <= 0 || K <= 0 ? 1 : plan_gated(M, F, K * element_bytes).splits;
}

extern "C" int fla_gated_linear_fwd(const void* x, const void* gate_weight, const void* up_weight, const void* gate_bias, const void* up_bias,
                                    int bias_dtype, void* h, float* gate_out, float* up_out, int64_t ld, int64_t M, int64_t F, int64_t K,
                                    int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && gate_weight && up_weight && h && (!gate_out == !up_out) && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!gate_bias && !up_bias) || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!gate_out || (ld >= F && ld % 8 == 0 && ld < F + 8), FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, gate_weight, up_weight, gate_out, up_out, workspace}) && aligned4({gate_bias, up_bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedParams p{};
  p.x = (const char*)x, p.wg = (const char*)gate_weight, p.wu = (const char*)up_weight, p.bg = gate_bias, p.bu = up_bias, p.h = h;
  p.g = gate_out, p.u = up_out, p.part = workspace, p.M = M, p.F = F, p.K = K, p.ldk = gate_out ? ld : (F + 7) / 8 * 8;
  p.act = activation, p.bias_f32 = bias_dtype == FLA_F32;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? gated_forward<bf16, bf16>(p, st) : fla_gated_linear_f16(&p, st);
}
