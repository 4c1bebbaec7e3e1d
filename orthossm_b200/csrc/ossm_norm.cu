// Entry points of the residual with norms: argument checks, and the choice of
// the types' kernels (a file each, ossm_norm_*.cu).
#include "ossm_norm.cuh"

namespace ossm {
namespace nrm {

typedef __nv_bfloat16 bf;
typedef __half hf;
#define OSSM_NORM_TYPES(TX, TY)                                \
  extern template int forward<TX, TY>(const ossm_norm_args*, cudaStream_t); \
  extern template int backward<TX, TY>(const ossm_norm_args*, const Plan&, float*, cudaStream_t);
OSSM_NORM_TYPES(float, float)
OSSM_NORM_TYPES(bf, bf)
OSSM_NORM_TYPES(hf, hf)
OSSM_NORM_TYPES(float, bf)
OSSM_NORM_TYPES(float, hf)
#undef OSSM_NORM_TYPES

bool float_type(int t) { return t == OSSM_F32 || t == OSSM_BF16 || t == OSSM_F16; }

bool valid(const ossm_norm_args* a, bool bwd) {
  if (!a || a->tokens < 0 || a->tokens > (1LL << 31) - 1 || a->dim < 1 || a->dim > 8192) return false;
  if (!float_type(a->stream_dtype) || !float_type(a->dtype)) return false;
  if (a->stream_dtype != a->dtype && a->stream_dtype != OSSM_F32) return false;
  if (a->norm < OSSM_NORM_RMS || a->norm > OSSM_NORM_LAYER || a->post_norm < OSSM_NORM_NONE || a->post_norm > OSSM_NORM_LAYER)
    return false;
  if (a->gate_kind < OSSM_GATE_NONE || a->gate_kind > OSSM_GATE_FULL || (a->gate_kind && !a->gate)) return false;
  if (!(a->eps >= 0.f) || !(a->post_eps >= 0.f) || !std::isfinite(a->eps) || !std::isfinite(a->post_eps)) return false;
  if (!std::isfinite(a->scale)) return false;
  if ((a->weight && !float_type(a->weight_dtype)) || (a->bias && !float_type(a->bias_dtype)) ||
      (a->post_weight && !float_type(a->post_weight_dtype)) || (a->post_bias && !float_type(a->post_bias_dtype)) ||
      (a->gate_kind && !float_type(a->gate_dtype)))
    return false;
  if (!a->y && (a->post_norm || a->gate_kind)) return false;
  if (!a->post_norm && (a->post_weight || a->post_bias)) return false;
  if (a->gate_kind == OSSM_GATE_FULL && a->gate_stride < a->dim) return false;
  if (!a->tokens) return true;
  const bool full = a->post_norm || a->gate_kind;
  if (!bwd) {
    if (!a->x || a->x_stride < a->dim || !a->h || (a->y && (a->y_stride < a->dim || !a->r))) return false;
    return true;
  }
  if (!a->stats) return false;
  if (a->x_stride < a->dim || (full && !a->y)) return false;
  if (a->y ? (!a->x || a->y_stride < a->dim) : !a->r) return false;
  if ((a->grad_r && a->grad_r_stride < a->dim) || (a->grad_h && a->grad_h_stride < a->dim)) return false;
  return a->grad_r || a->grad_h;
}

template <typename F>
int by_type(const ossm_norm_args* a, F f) {
  if (a->stream_dtype == OSSM_BF16) return f((bf*)nullptr, (bf*)nullptr);
  if (a->stream_dtype == OSSM_F16) return f((hf*)nullptr, (hf*)nullptr);
  if (a->dtype == OSSM_BF16) return f((float*)nullptr, (bf*)nullptr);
  if (a->dtype == OSSM_F16) return f((float*)nullptr, (hf*)nullptr);
  return f((float*)nullptr, (float*)nullptr);
}

}  // namespace nrm
}  // namespace ossm

using namespace ossm;

extern "C" size_t ossm_norm_workspace_bytes(const ossm_norm_args* a) {
  return nrm::valid(a, true) ? std::max<size_t>(256, nrm::plan_of(a, true).bytes) : 0;
}
extern "C" int ossm_residual_norm_fwd(const ossm_norm_args* a, ossm_stream_t stream) {
  if (!nrm::valid(a, false)) return OSSM_EINVAL;
  if (!a->tokens) return OSSM_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return nrm::by_type(a, [&](auto* x, auto* y) {
    return nrm::forward<std::remove_pointer_t<decltype(x)>, std::remove_pointer_t<decltype(y)>>(a, st);
  });
}
extern "C" int ossm_residual_norm_bwd(const ossm_norm_args* a, void* workspace, size_t workspace_bytes,
                                      ossm_stream_t stream) {
  if (!nrm::valid(a, true)) return OSSM_EINVAL;
  const nrm::Plan q = nrm::plan_of(a, true);
  if (!workspace || workspace_bytes < q.bytes || (uintptr_t)workspace % 256) return OSSM_EWORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return nrm::by_type(a, [&](auto* x, auto* y) {
    return nrm::backward<std::remove_pointer_t<decltype(x)>, std::remove_pointer_t<decltype(y)>>(
        a, q, static_cast<float*>(workspace), st);
  });
}
extern "C" size_t ossm_sizeof_norm_args(void) { return sizeof(ossm_norm_args); }
