// The product kernel on float16 operands.
#include "linear.h"

int lin_launch_f16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinF16, dl_f16>(g, p, turn_a, turn_b, gated, s);
}
