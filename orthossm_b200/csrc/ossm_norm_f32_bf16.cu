// The residual with norms, an fp32 stream beside bf16.
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {
template int forward<float, __nv_bfloat16>(const ossm_norm_args*, cudaStream_t);
template int backward<float, __nv_bfloat16>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
}  // namespace nrm
}  // namespace ossm
