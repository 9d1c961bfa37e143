// xent_few_bf16.cu -- the few-class cross entropy kernels (xent_few.cuh) of bf16 tables.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_bf16(const FewPlan& p, cudaStream_t s) { return few::launch_t<__nv_bfloat16>(p, s); }

}  // namespace gafime
