// The product kernel on bfloat16 operands.
#include "linear.h"

int lin_launch_bf16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinBf16, dl_bf16>(g, p, turn_a, turn_b, gated, s);
}
