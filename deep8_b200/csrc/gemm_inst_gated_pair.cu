// Instantiation of the paired-CTA gated fp16 kernel: 256 x 128 outputs per pair.
#include "gemm2_kernel.cuh"
#include "gemm_host.h"

namespace d8k {

GemmLaunchFn lookup_f16_gated_pair() { return launch_pair_cfg<Gemm2Cfg<false, true, 3, 2, true>>; }

}  // namespace d8k
