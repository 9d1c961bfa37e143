// xent_few_bf16_columns.cu -- the few-class cross entropy kernels (xent_few.cuh) of bf16 tables by columns.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, __nv_bfloat16) { return few::launch_t<__nv_bfloat16, true>(p, s); }

}  // namespace gafime
