// The float16 kernels of the channels-last group norm (group_norm.cuh).
#include "group_norm.cuh"

namespace actnn {
int gn_run_f16(const GnCall& c, const GnShape& g, bool forward) { return gn_run<__half>(c, g, forward); }
}  // namespace actnn
