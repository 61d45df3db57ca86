// The product kernel on float16 operands: forward, small tiles.
#include "linear.h"

LIN_TILE(LinF16, dl_f16, 128, false, false);
