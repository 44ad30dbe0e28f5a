// Products of rows in 8-bit integers with results in fp16.
#include "int8_linear.h"

int fla_int8_linear_f16(void* p, hipStream_t st) { return launch_int8<f16>(*(Int8Params*)p, st); }
