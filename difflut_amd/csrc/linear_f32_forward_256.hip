// The product kernel on float32 (as bf16 planes) operands: forward, large tiles.
#include "linear.h"

LIN_TILE(LinF32, float, 256, false, false);
