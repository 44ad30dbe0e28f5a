// The gated product of fp16 rows.
#include "gated_forward.h"

int fla_gated_linear_f16(void* p, hipStream_t st) { return gated_forward<f16, f16>(*(GatedParams*)p, st); }
