// The residual with norms, fp32.
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {
template int forward<float, float>(const ossm_norm_args*, cudaStream_t);
template int backward<float, float>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
}  // namespace nrm
}  // namespace ossm
