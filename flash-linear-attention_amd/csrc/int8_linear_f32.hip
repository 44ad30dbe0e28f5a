// Products of rows in 8-bit integers with results in fp32.
#include "int8_linear.h"

int fla_int8_linear_f32(void* p, hipStream_t st) { return launch_int8<float>(*(Int8Params*)p, st); }
