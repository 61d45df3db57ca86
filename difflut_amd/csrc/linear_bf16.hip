// Launches of the product kernel on bfloat16 operands.
#include "linear.h"

extern LIN_TILE(LinBf16, dl_bf16, 256, false, false);
extern LIN_TILE(LinBf16, dl_bf16, 128, false, false);
extern LIN_TILE(LinBf16, dl_bf16, 256, false, true);
extern LIN_TILE(LinBf16, dl_bf16, 128, false, true);
extern LIN_TILE(LinBf16, dl_bf16, 256, true, true);
extern LIN_TILE(LinBf16, dl_bf16, 128, true, true);

int lin_launch_bf16(LinArgs &g, const LinPlan &p, bool turn_a, bool turn_b, bool gated, hipStream_t s) {
    return lin_launch_turned<LinBf16, dl_bf16>(g, p, turn_a, turn_b, gated, s);
}
