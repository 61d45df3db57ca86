// The product kernel on 8-bit operands, results in float16.
#include "linear.h"

LIN_TILE(LinE4m3, dl_f16, 256, false, false);
LIN_TILE(LinE4m3, dl_f16, 128, false, false);
