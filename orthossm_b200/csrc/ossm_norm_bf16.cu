// The residual with norms, bf16.
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {
template int forward<__nv_bfloat16, __nv_bfloat16>(const ossm_norm_args*, cudaStream_t);
template int backward<__nv_bfloat16, __nv_bfloat16>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
}  // namespace nrm
}  // namespace ossm
