// xent_few_fp16.cu -- the few-class cross entropy kernels (xent_few.cuh) of fp16 tables.
#include "xent_few.cuh"

namespace gafime {

cudaError_t few_launch_fp16(const FewPlan& p, cudaStream_t s) { return few::launch_t<__half>(p, s); }

}  // namespace gafime
