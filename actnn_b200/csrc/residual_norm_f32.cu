// The float32 kernels of the norms around a residual branch (residual_norm.cuh).
#include "residual_norm.cuh"

namespace actnn {
int rn_run_f32(const RnArgs& a, RnWhat what, bool vec) { return rn_run<float>(a, what, vec); }
}  // namespace actnn
