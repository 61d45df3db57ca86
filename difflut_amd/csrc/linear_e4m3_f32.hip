// The product kernel on 8-bit operands, results in float32.
#include "linear.h"

LIN_TILE(LinE4m3, float, 256, false, false);
LIN_TILE(LinE4m3, float, 128, false, false);
