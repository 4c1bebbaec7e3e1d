// The norms' kernels with waits that run out at once, for a test of what they
// leave: no polls of a row's barrier, the copies themselves as they are.
#define OSSM_NORM_POLLS 0u
#include "ossm_norm.cuh"

namespace ossm {
int device_sms() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}
}  // namespace ossm
using namespace ossm;
using namespace ossm::nrm;
typedef __nv_bfloat16 bf;

template <typename K>
static int launch(K kern, const Params& p, const Plan& q, size_t smem, cudaStream_t st) {
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes) != cudaSuccess) return 1;
  kern<<<q.blocks, q.R * q.per, smem, st>>>(p);
  return cudaGetLastError() != cudaSuccess;
}

// bf16 rows of 257 to 4096 channels, whole 16-byte pieces.
extern "C" int norm_wait_fwd(const ossm_norm_args* a, cudaStream_t st) {
  const Plan q = plan_of(a, false);
  Params p = params_of(a, q, false);
  const size_t smem = ring_of(p, q, false, 2 * p.d * (a->y ? 2 : 1));
  if (!p.vec || q.N != 2 || q.R > 256) return 2;
  return launch(norm_fwd_kernel<bf, bf, 2, true, 256>, p, q, smem, st);
}
// A weight's gradient, or all sums; part: room for plan's blocks.
extern "C" size_t norm_wait_bytes(const ossm_norm_args* a) { return plan_of(a, true).bytes; }
extern "C" int norm_wait_bwd(const ossm_norm_args* a, float* part, cudaStream_t st) {
  const Plan q = plan_of(a, true);
  Params p = params_of(a, q, true);
  const size_t smem = ring_of(p, q, true, 2 * p.d * (1 + (p.dr != nullptr) + (p.dh != nullptr) + (p.y != nullptr)));
  p.part = part;
  if (!p.vec || q.R > 256 || (q.sums != 1 && q.sums != (int)kSums)) return 2;
  if (q.sums == 1)
    return q.N == 1 ? launch(norm_bwd_kernel<bf, bf, 1, true, 1, 256>, p, q, smem, st)
                    : launch(norm_bwd_kernel<bf, bf, 2, true, 1, 256>, p, q, smem, st);
  if (q.N != 1) return 2;
  return launch(norm_bwd_kernel<bf, bf, 1, true, (int)kSums, 256>, p, q, smem, st);
}
