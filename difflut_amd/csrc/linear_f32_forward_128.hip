// The product kernel on float32 (as bf16 planes) operands: forward, small tiles.
#include "linear.h"

LIN_TILE(LinF32, float, 128, false, false);
