// The product kernel on float32 (as bf16 planes) operands.
#include "linear.h"

int lin_launch_f32(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinF32, float>(g, p, turn_a, turn_b, gated, s);
}
