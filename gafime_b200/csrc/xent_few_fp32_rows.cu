// xent_few_fp32_rows.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp32 tables by rows.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, float) { return few::launch_t<float, false>(p, s); }

}  // namespace gafime
