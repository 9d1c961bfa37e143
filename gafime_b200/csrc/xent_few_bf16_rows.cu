// xent_few_bf16_rows.cu -- the few-class cross entropy kernels (xent_few.cuh) of bf16 tables by rows.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, __nv_bfloat16) { return few::launch_t<__nv_bfloat16, false>(p, s); }

}  // namespace gafime
