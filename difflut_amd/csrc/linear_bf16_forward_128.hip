// The product kernel on bfloat16 operands: forward, small tiles.
#include "linear.h"

LIN_TILE(LinBf16, dl_bf16, 128, false, false);
