// Launches of the product kernel on float16 operands.
#include "linear.h"

extern LIN_TILE(LinF16, dl_f16, 256, false, false);
extern LIN_TILE(LinF16, dl_f16, 128, false, false);
extern LIN_TILE(LinF16, dl_f16, 256, false, true);
extern LIN_TILE(LinF16, dl_f16, 128, false, true);
extern LIN_TILE(LinF16, dl_f16, 256, true, true);
extern LIN_TILE(LinF16, dl_f16, 128, true, true);

int lin_launch_f16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinF16, dl_f16>(g, p, turn_a, turn_b, gated, s);
}
