// xent_few_fp16_rows.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp16 tables by rows.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, __half) { return few::launch_t<__half, false>(p, s); }

}  // namespace gafime
