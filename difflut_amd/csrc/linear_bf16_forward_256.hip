// The product kernel on bfloat16 operands: forward, large tiles.
#include "linear.h"

LIN_TILE(LinBf16, dl_bf16, 256, false, false);
