// The product kernel on float16 operands: forward, large tiles.
#include "linear.h"

LIN_TILE(LinF16, dl_f16, 256, false, false);
