// The product kernel on float16 operands: backward.
#include "linear.h"

LIN_TILE(LinF16, dl_f16, 256, false, true);
LIN_TILE(LinF16, dl_f16, 128, false, true);
LIN_TILE(LinF16, dl_f16, 256, true, true);
LIN_TILE(LinF16, dl_f16, 128, true, true);
