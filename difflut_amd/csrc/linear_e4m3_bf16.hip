// The product kernel on 8-bit operands, results in bfloat16.
#include "linear.h"

LIN_TILE(LinE4m3, dl_bf16, 256, false, false);
LIN_TILE(LinE4m3, dl_bf16, 128, false, false);
