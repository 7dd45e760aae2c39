// The float16 kernels of the channels-last group norm (group_norm.cuh).
#include "group_norm.cuh"

namespace actnn {
int gn_forward_f16(const GnCall& c, const GnShape& g) { return gn_forward_of<__half>(c, g); }
int gn_backward_f16(const GnCall& c, const GnShape& g) { return gn_backward_of<__half>(c, g); }
}  // namespace actnn
