// RMS norm, and rows brought to 8 bits without a norm: the kernels of norm_rows.h without a mean.
#include "norm_rows.h"

extern "C" int fla_rms_norm_rows8_fwd(const void* x, const void* residual, int residual_dtype, const void* weight, const void* bias,
                                      int weight_dtype, void* y, float* scale, void* residual_out, int residual_out_dtype, int64_t M,
                                      int64_t N, float eps, int normalise, int rows8, int dtype, fla_stream_t stream) {
  return norm_forward<false>(x, residual, residual_dtype, weight, bias, weight_dtype, y, scale, residual_out, residual_out_dtype, nullptr,
                             nullptr, M, N, eps, normalise, rows8, dtype, stream);
}

extern "C" int fla_rms_norm_fwd(const void* x, const void* residual, int residual_dtype, const void* weight, const void* bias,
                                int weight_dtype, void* y, float* scale, void* residual_out, int residual_out_dtype, float* rstd,
                                int64_t M, int64_t N, float eps, int normalise, int dtype, fla_stream_t stream) {
  return norm_forward<false>(x, residual, residual_dtype, weight, bias, weight_dtype, y, scale, residual_out, residual_out_dtype, nullptr,
                             rstd, M, N, eps, normalise, scale ? FLA_ROWS_E4M3 : FLA_ROWS_NONE, dtype, stream);
}

extern "C" int fla_rms_norm_workgroups(int64_t M, int64_t N) { return norm_workgroups(M, N); }

extern "C" int fla_rms_norm_bwd(const void* dy, const void* kept, int kept_dtype, const void* weight, int weight_dtype, const float* rstd,
                                const void* dresidual, void* dx, void* dresidual_in, float* dw_partial, float* db_partial, int64_t M,
                                int64_t N, int dtype, fla_stream_t stream) {
  FLA_REQUIRE(((uintptr_t)dw_partial | (uintptr_t)db_partial) % 16 == 0, FLA_E_ALIGNMENT);
  return norm_backward<false>(dy, kept, kept_dtype, weight, weight_dtype, nullptr, rstd, dresidual, dx, dresidual_in, dw_partial, db_partial, N,
                              M, N, dtype, stream);
}
