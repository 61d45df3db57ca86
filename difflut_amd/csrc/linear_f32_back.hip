// The product kernel on float32 (as bf16 planes) operands: backward.
#include "linear.h"

LIN_TILE(LinF32, float, 256, false, true);
LIN_TILE(LinF32, float, 128, false, true);
LIN_TILE(LinF32, float, 256, true, true);
LIN_TILE(LinF32, float, 128, true, true);
