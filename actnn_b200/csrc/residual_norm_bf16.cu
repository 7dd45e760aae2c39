// The bfloat16 kernels of the norms around a residual branch (residual_norm.cuh).
#include "residual_norm.cuh"

namespace actnn {
int rn_run_bf16(const RnArgs& a, RnWhat what, bool vec) { return rn_run<__nv_bfloat16>(a, what, vec); }
}  // namespace actnn
