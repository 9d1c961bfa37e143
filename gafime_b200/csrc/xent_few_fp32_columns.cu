// xent_few_fp32_columns.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp32 tables by columns.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, float) { return few::launch_t<float, true>(p, s); }

}  // namespace gafime
