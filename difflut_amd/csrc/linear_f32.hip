// Launches of the product kernel on float32 (as bf16 planes) operands.
#include "linear.h"

extern LIN_TILE(LinF32, float, 256, false, false);
extern LIN_TILE(LinF32, float, 128, false, false);
extern LIN_TILE(LinF32, float, 256, false, true);
extern LIN_TILE(LinF32, float, 128, false, true);
extern LIN_TILE(LinF32, float, 256, true, true);
extern LIN_TILE(LinF32, float, 128, true, true);

int lin_launch_f32(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinF32, float>(g, p, turn_a, turn_b, gated, s);
}
