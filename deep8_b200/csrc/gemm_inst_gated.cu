// Instantiations of the gated kernels: act(A B[0]) * (A B[1]) with A K-major and the two projections MN-major.
#include "gemm_host.h"

namespace d8k {

// fp16 behind TMA with twin issuing threads (GemmCfg::TWIN): 128 or 64 output columns per tile
GemmLaunchFn lookup_f16_gated(int bn) {
    if (bn == 256) return launch_cfg<GemmCfg<false, false, true, 256, 4, false, false, false, 4, true>>;
    if (bn == 128) return launch_cfg<GemmCfg<false, false, true, 128, 6, false, false, false, 4, true>>;
    return nullptr;
}

// fp32 (3xTF32) behind TMA, 32 output columns per tile: two CTAs per SM (modes 1 and 2) or twin issuing threads (mode 4)
GemmLaunchFn lookup_f32_gated(int mode) {
    if (mode == 4) return launch_cfg<GemmCfg<true, false, true, 64, 4, false, true, false, 4, true>>;
    if (mode == 2) return launch_cfg<GemmCfg<true, false, true, 64, 3, false, true, false, 2, true>>;
    return launch_cfg<GemmCfg<true, false, true, 64, 2, false, true, false, 1, true>>;
}

GemmLaunchFn lookup_gated_gather(bool f32) {
    if (f32) return launch_cfg<GemmCfg<true, false, true, 64, 4, true, false, false, 0, true>>;
    return launch_cfg<GemmCfg<false, false, true, 128, 6, true, false, false, 0, true>>;
}

}  // namespace d8k
