// xent_few_fp32.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp32 tables.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_fp32(const FewPlan& p, cudaStream_t s) { return few::launch_t<float>(p, s); }

}  // namespace gafime
