// The residual with norms, an fp32 stream beside fp16.
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {
template int forward<float, __half>(const ossm_norm_args*, cudaStream_t);
template int backward<float, __half>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
}  // namespace nrm
}  // namespace ossm
