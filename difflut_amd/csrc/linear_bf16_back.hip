// The product kernel on bfloat16 operands: backward.
#include "linear.h"

LIN_TILE(LinBf16, dl_bf16, 256, false, true);
LIN_TILE(LinBf16, dl_bf16, 128, false, true);
LIN_TILE(LinBf16, dl_bf16, 256, true, true);
LIN_TILE(LinBf16, dl_bf16, 128, true, true);
