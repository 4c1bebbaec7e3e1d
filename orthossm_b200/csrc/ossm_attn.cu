// Entry points of the attention over packed prompts or over a cache: argument
// checks, workspace, and the choice between the kernels for many and for few
// queries a sequence.
#include <algorithm>
#include <cmath>

#include "ossm_attn.cuh"

namespace ossm {
int device_sms();
namespace attn {

size_t prompt_part_floats(int hd);
int prompt_forward(const ossm_attn_args* a, const Params& p, int grid, cudaStream_t st);
size_t token_part_floats(int hd);
int token_forward(const ossm_attn_args* a, const Params& p, int sms, cudaStream_t st);

bool row_ok(const void* ptr, long long st, long long sh, long long rows, int heads) {
  return ptr && (uintptr_t)ptr % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && (rows <= 1 || st > 0) &&
         (heads <= 1 || sh > 0);
}

bool valid(const ossm_attn_args* a) {
  if (!a || a->B < 1 || a->B > kMaxSeqs || a->H < 1 || a->H_kv < 1 || a->H % a->H_kv || a->H > 65535) return false;
  if (a->head_dim < 8 || a->head_dim > kMaxHD || a->head_dim % 8) return false;
  if (a->total_q < 0 || a->total_k < 0 || a->total_q > kMaxRows || a->total_k > kMaxRows ||
      a->total_q * a->H > 0x7fffffffLL)
    return false;
  if (a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) return false;
  if (a->flags & ~OSSM_ATTN_NO_CAPTURE) return false;
  if (a->window < 0 || !(a->scale > 0.f) || !std::isfinite(a->scale * 1.5f) || !a->cu_q || !a->cu_k) return false;
  if (a->total_q == 0) return true;
  if (!row_ok(a->q, a->q_stride_t, a->q_stride_h, a->total_q, a->H) ||
      !row_ok(a->out, a->out_stride_t, a->out_stride_h, a->total_q, a->H))
    return false;
  return a->total_k == 0 || (row_ok(a->k, a->k_stride_t, a->k_stride_h, a->total_k, a->H_kv) &&
                             row_ok(a->v, a->v_stride_t, a->v_stride_h, a->total_k, a->H_kv));
}

}  // namespace attn
}  // namespace ossm

using namespace ossm;

// SMs of the current device (asked for once a device).
int ossm::device_sms() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

namespace {

// Workspace: header, progress counters, two partial results a CTA.
constexpr int kTokenRows = 16;  // of the token kernel's items

int sm_count() { return std::min(device_sms(), attn::kMaxSms); }

// One size for all arguments: a workspace never has to be replaced by a larger
// one while a captured graph still points to it.
size_t ws_bytes() {
  size_t part = 0;
  for (int hd : {64, attn::kMaxHD})
    part = std::max({part, attn::prompt_part_floats(hd), attn::token_part_floats(hd)});
  return sizeof(WsHeader) + attn::kCounters * sizeof(uint32_t) + (size_t)sm_count() * part * sizeof(float);
}
static_assert(sizeof(WsHeader) + attn::kCounters * sizeof(uint32_t) <= OSSM_ATTN_WS_ZERO, "header and counters");

}  // namespace

extern "C" size_t ossm_attn_workspace_bytes(const ossm_attn_args* a) { return attn::valid(a) ? ws_bytes() : 0; }

extern "C" int ossm_attention_fwd(const ossm_attn_args* a, void* workspace, size_t workspace_bytes,
                                  ossm_stream_t stream) {
  if (!attn::valid(a)) return OSSM_EINVAL;
  if (!workspace || workspace_bytes < ws_bytes() || (uintptr_t)workspace % 256) return OSSM_EWORKSPACE;
  if (a->total_q == 0) return OSSM_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->flags & OSSM_ATTN_NO_CAPTURE) {
    cudaStreamCaptureStatus on = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &on) != cudaSuccess) return OSSM_ELAUNCH;
    if (on != cudaStreamCaptureStatusNone) return OSSM_EWORKSPACE;
  }
  char* w = static_cast<char*>(workspace);
  const attn::Params p{a->B, a->H, a->H_kv, a->head_dim, (int)a->total_q, (int)a->total_k, a->q, a->k, a->v, a->out,
                       a->q_stride_t, a->q_stride_h, a->k_stride_t, a->k_stride_h, a->v_stride_t, a->v_stride_h,
                       a->out_stride_t, a->out_stride_h, a->cu_q, a->cu_k, a->kv_len,
                       a->window >= a->total_k ? 0 : a->window,  // as wide as all keys: none
                       a->scale * 1.4426950408889634f, reinterpret_cast<WsHeader*>(w),
                       reinterpret_cast<uint32_t*>(w + sizeof(WsHeader)),
                       reinterpret_cast<float*>(w + sizeof(WsHeader) + attn::kCounters * sizeof(uint32_t))};
  // Rows that share a key head.  Up to 16, one item of the token kernel holds
  // them and K and V are read once (8 streams of 2000 keys, 8/8 heads of 128,
  // 16 new tokens: 23 us, 28 us on the prompt kernel; 32 of 8192, 32/8 of 128,
  // 1 token: 167 and 180 us; 64 of 1000, 16/4 of 64, 1 token: 19 and 34 us).
  // Up to 32 they are read twice, which still pays at 64 channels (32 of 8192,
  // 8/8 of 64, 32 tokens: 133 and 160 us; 64 of 1000, 16/4, 8: 31 and 34 us) and
  // not above (8 of 2000, 8/8 of 128, 32 tokens: 31 and 28 us; 32 of 8192, 32/8
  // of 128, 8: 330 and 187 us).  Beyond, the prompt kernel's tile of 128 rows.
  const int64_t rows = (int64_t)a->max_seqlen_q * (a->H / a->H_kv);
  if (a->total_k == 0 || rows <= (a->head_dim <= 64 ? 2 : 1) * kTokenRows)
    return attn::token_forward(a, p, sm_count(), st);
  return attn::prompt_forward(a, p, sm_count(), st);
}
