// The bfloat16 kernels of the channels-last group norm (group_norm.cuh).
#include "group_norm.cuh"

namespace actnn {
int gn_forward_bf16(const GnCall& c, const GnShape& g) { return gn_forward_of<__nv_bfloat16>(c, g); }
int gn_backward_bf16(const GnCall& c, const GnShape& g) { return gn_backward_of<__nv_bfloat16>(c, g); }
}  // namespace actnn
