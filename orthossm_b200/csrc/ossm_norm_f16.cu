// The residual with norms, fp16.
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {
template int forward<__half, __half>(const ossm_norm_args*, cudaStream_t);
template int backward<__half, __half>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
}  // namespace nrm
}  // namespace ossm
