// Launches of the product kernel on 8-bit operands.
#include "linear.h"

extern LIN_TILE(LinE4m3, float, 256, false, false);
extern LIN_TILE(LinE4m3, float, 128, false, false);
extern LIN_TILE(LinE4m3, dl_bf16, 256, false, false);
extern LIN_TILE(LinE4m3, dl_bf16, 128, false, false);
extern LIN_TILE(LinE4m3, dl_f16, 256, false, false);
extern LIN_TILE(LinE4m3, dl_f16, 128, false, false);

int lin_launch_e4m3(LinArgs &g, const LinPlan &p, int out_type, bool gated, hipStream_t s) {
    int code = DL_ERR_UNSUPPORTED;
    DL_BY_TYPE(out_type, Out, (code = p.few ? lin_launch_few<LinE4m3, Out>(g, gated, s) : lin_launch<LinE4m3, Out, false, false>(g, p, gated, s)));
    return code;
}
