// Attention over packed prompts or over a cache (ossm_attention_fwd).
//
// One warp per (query, head): the softmax over its keys with a running
// maximum and sum, 32 keys at a time (a lane's key each for the scores, a
// lane's channels each for the weighted sum).
#include <algorithm>
#include <cmath>

#include "ossm_attn.cuh"

namespace ossm {
namespace attn {

size_t prompt_part_floats(int hd);
int prompt_forward(const ossm_attn_args* a, const Params& p, int grid, cudaStream_t st);

template <typename T>
__global__ void __launch_bounds__(128) attn_rows_kernel(const Params p) {
  __shared__ float qs[4][kMaxHD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + warp, h = blockIdx.y;
  if (t >= p.Tq) return;
  int lo = 0, hi = p.B;  // the last b with cu_q[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.cu_q + mid) <= t) lo = mid; else hi = mid;
  }
  const Seq s = seq_of(p, lo);
  const int i = t - s.q0;
  if (i < 0 || i >= s.nq) return;
  const T* q = static_cast<const T*>(p.q) + t * p.qst + h * p.qsh;
  const int hk = h / (p.H / p.Hkv);
  const T* k = static_cast<const T*>(p.k) + s.k0 * p.kst + hk * p.ksh;
  const T* v = static_cast<const T*>(p.v) + s.k0 * p.vst + hk * p.vsh;
  for (int d = lane; d < p.hd; d += 32) qs[warp][d] = (float)q[d] * p.scale2;
  __syncwarp();
  const int at = i + s.nk - s.nq;
  const int end = min(at + 1, s.nk), begin = p.window ? max(0, at - p.window + 1) : 0;
  float m = -INFINITY, l = 0.f, o[kMaxHD / 32] = {};
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    if (j < end) {
      x = 0.f;
      for (int d = 0; d < p.hd; d += 2) {
        const float2 kv = to_f2<T>(*reinterpret_cast<const uint32_t*>(k + j * p.kst + d));
        x = fmaf(kv.x, qs[warp][d], fmaf(kv.y, qs[warp][d + 1], x));
      }
    }
    float mx = x;
    for (int w = 16; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, w));
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(m - ms), w = j < end ? ex2(x - ms) : 0.f;
    m = mn;
    l = l * f + w;
    for (int c = 0; c < kMaxHD / 32; ++c) o[c] *= f;
    const int n = min(32, end - j0);
    for (int jj = 0; jj < n; ++jj) {
      const float pj = __shfl_sync(~0u, w, jj);
      const T* vr = v + (j0 + jj) * p.vst;
      for (int c = 0; c < kMaxHD / 32; ++c)
        if (c * 32 + lane < p.hd) o[c] = fmaf(pj, (float)vr[c * 32 + lane], o[c]);
    }
  }
  for (int w = 16; w; w >>= 1) l += __shfl_xor_sync(~0u, l, w);
  const float inv = end > begin ? 1.f / l : 0.f;
  T* out = static_cast<T*>(p.out) + t * p.ost + h * p.osh;
  for (int c = 0; c < kMaxHD / 32; ++c)
    if (c * 32 + lane < p.hd) out[c * 32 + lane] = T(o[c] * inv);
}

bool row_ok(const void* ptr, long long st, long long sh, long long rows, int heads) {
  return ptr && (uintptr_t)ptr % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && (rows <= 1 || st > 0) &&
         (heads <= 1 || sh > 0);
}

bool valid(const ossm_attn_args* a) {
  if (!a || a->B < 1 || a->B > kMaxSeqs || a->H < 1 || a->H_kv < 1 || a->H % a->H_kv || a->H > 65535) return false;
  if (a->head_dim < 8 || a->head_dim > kMaxHD || a->head_dim % 8) return false;
  if (a->total_q < 0 || a->total_k < 0 || a->total_q > kMaxRows || a->total_k > kMaxRows) return false;
  if (a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) return false;
  if (a->window < 0 || !(a->scale > 0.f) || !std::isfinite(a->scale) || !a->cu_q || !a->cu_k) return false;
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

namespace {

// Workspace: header, two progress counters a CTA, two partial results a CTA.
constexpr int kMaxCtas = 1024;

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return std::min(n, kMaxCtas);
}

size_t ws_bytes(const ossm_attn_args* a) {
  return sizeof(WsHeader) + 2 * kMaxCtas * sizeof(uint32_t) + (size_t)sm_count() * attn::prompt_part_floats(a->head_dim) * 4;
}

}  // namespace

extern "C" size_t ossm_attn_workspace_bytes(const ossm_attn_args* a) { return attn::valid(a) ? ws_bytes(a) : 0; }

extern "C" int ossm_attention_fwd(const ossm_attn_args* a, void* workspace, size_t workspace_bytes,
                                  ossm_stream_t stream) {
  if (!attn::valid(a)) return OSSM_EINVAL;
  if (!workspace || workspace_bytes < ws_bytes(a) || (uintptr_t)workspace % 256) return OSSM_EWORKSPACE;
  if (a->total_q == 0) return OSSM_OK;
  char* w = static_cast<char*>(workspace);
  const attn::Params p{a->B, a->H, a->H_kv, a->head_dim, (int)a->total_q, (int)a->total_k, a->q, a->k, a->v, a->out,
                       a->q_stride_t, a->q_stride_h, a->k_stride_t, a->k_stride_h, a->v_stride_t, a->v_stride_h,
                       a->out_stride_t, a->out_stride_h, a->cu_q, a->cu_k, a->kv_len,
                       a->window >= a->total_k ? 0 : a->window,  // as wide as all keys: none
                       a->scale * 1.4426950408889634f, reinterpret_cast<WsHeader*>(w),
                       reinterpret_cast<uint32_t*>(w + sizeof(WsHeader)),
                       reinterpret_cast<float*>(w + sizeof(WsHeader) + 2 * kMaxCtas * sizeof(uint32_t))};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->max_seqlen_q > 16 && a->total_k > 0) return attn::prompt_forward(a, p, sm_count(), st);
  const dim3 grid((unsigned)((a->total_q + 3) / 4), a->H);
  if (a->dtype == OSSM_BF16)
    attn::attn_rows_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(p);
  else
    attn::attn_rows_kernel<__half><<<grid, 128, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}
