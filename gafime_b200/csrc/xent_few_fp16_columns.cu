// xent_few_fp16_columns.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp16 tables by columns.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, __half) { return few::launch_t<__half, true>(p, s); }

}  // namespace gafime
