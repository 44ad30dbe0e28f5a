// Layer norm: the kernels of norm_rows.h with a mean.
#include "norm_rows.h"

extern "C" int fla_layer_norm_fwd(const void* x, const void* residual, int residual_dtype, const void* weight, const void* bias,
                                  int weight_dtype, void* y, float* scale, void* residual_out, int residual_out_dtype, float* mean,
                                  float* rstd, int64_t M, int64_t N, float eps, int rows8, int dtype, fla_stream_t stream) {
  return norm_forward<true>(x, residual, residual_dtype, weight, bias, weight_dtype, y, scale, residual_out, residual_out_dtype, mean, rstd, M,
                            N, eps, 1, rows8, dtype, stream);
}

extern "C" int fla_layer_norm_workgroups(int64_t M, int64_t N) { return norm_workgroups(M, N); }

extern "C" int fla_layer_norm_bwd(const void* dy, const void* kept, int kept_dtype, const void* weight, int weight_dtype, const float* mean,
                                  const float* rstd, const void* dresidual, void* dx, void* dresidual_in, float* dw_partial,
                                  float* db_partial, int64_t partial_ld, int64_t M, int64_t N, int dtype,
                                  fla_stream_t stream) {
  return norm_backward<true>(dy, kept, kept_dtype, weight, weight_dtype, mean, rstd, dresidual, dx, dresidual_in, dw_partial, db_partial,
                             partial_ld, M, N, dtype, stream);
}
