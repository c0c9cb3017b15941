// Instantiations of the fp32 kernels with short accumulation chains (GemmCfg::PRECISE) for the gated block's gradient products: two K-major operands
// (the gradient of x) or two MN-major ones (of w).
#include "gemm_host.h"

namespace d8k {

template <bool MN>
static GemmLaunchFn pick(int mode) {
    if (mode == 4) return launch_cfg<GemmCfg<true, MN, MN, 64, 4, false, true, false, 4, false, true>>;
    if (mode == 2) return launch_cfg<GemmCfg<true, MN, MN, 64, 3, false, true, false, 2, false, true>>;
    if (mode == 1) return launch_cfg<GemmCfg<true, MN, MN, 64, 2, false, true, false, 1, false, true>>;
    return launch_cfg<GemmCfg<true, MN, MN, 64, 4, true, false, false, 0, false, true>>;  // loader warps
}

GemmLaunchFn lookup_f32_precise(bool mn, int mode) { return mn ? pick<true>(mode) : pick<false>(mode); }

}  // namespace d8k
