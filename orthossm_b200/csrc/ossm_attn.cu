// Attention over packed prompts or over a cache (ossm_attention_fwd).
//
// One warp per (query, head): the softmax over its keys with a running
// maximum and sum, 32 keys at a time (a lane's key each for the scores, a
// lane's channels each for the weighted sum).
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "orthossm_b200.h"
#include "ossm_common.cuh"

namespace ossm {
namespace attn {

constexpr int kMaxSeqs = 16384;
constexpr int kMaxHD = 128;

struct Params {
  int B, H, Hkv, hd;
  int Tq, Tk;
  const void *q, *k, *v;
  void* out;
  long long qst, qsh, kst, ksh, vst, vsh, ost, osh;
  const int *cu_q, *cu_k, *kv_len;
  int window;
  float scale;
};

// The rows of sequence b, clipped to the tensors.
struct Seq {
  int q0, nq, k0, nk;
};
OSSM_DEV Seq seq_of(const Params& p, int b) {
  Seq s;
  s.q0 = min(max(__ldg(p.cu_q + b), 0), p.Tq);
  s.nq = min(max(__ldg(p.cu_q + b + 1), s.q0), p.Tq) - s.q0;
  s.k0 = min(max(__ldg(p.cu_k + b), 0), p.Tk);
  s.nk = min(max(__ldg(p.cu_k + b + 1), s.k0), p.Tk) - s.k0;
  if (p.kv_len) s.nk = min(s.nk, max(__ldg(p.kv_len + b), 0));
  return s;
}

template <typename T>
OSSM_DEV float2 to_f2(uint32_t u);
template <>
OSSM_DEV float2 to_f2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
OSSM_DEV float2 to_f2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}
template <typename T>
OSSM_DEV T from_f(float v);
template <>
OSSM_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
OSSM_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }

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
  for (int d = lane; d < p.hd; d += 32) qs[warp][d] = (float)q[d] * p.scale;
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
    const float f = __expf(m - ms), w = j < end ? __expf(x - ms) : 0.f;
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
    if (c * 32 + lane < p.hd) out[c * 32 + lane] = from_f<T>(o[c] * inv);
}

bool row_ok(const void* ptr, long long st, long long sh, long long rows, int heads) {
  return ptr && (uintptr_t)ptr % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && (rows <= 1 || st > 0) &&
         (heads <= 1 || sh > 0);
}

bool valid(const ossm_attn_args* a) {
  if (!a || a->B < 1 || a->B > kMaxSeqs || a->H < 1 || a->H_kv < 1 || a->H % a->H_kv || a->H > 65535) return false;
  if (a->head_dim < 8 || a->head_dim > kMaxHD || a->head_dim % 8) return false;
  if (a->total_q < 0 || a->total_k < 0 || a->total_q > 0x7fffffffLL || a->total_k > 0x7fffffffLL) return false;
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

extern "C" size_t ossm_attn_workspace_bytes(const ossm_attn_args* a) { return attn::valid(a) ? sizeof(WsHeader) : 0; }

extern "C" int ossm_attention_fwd(const ossm_attn_args* a, void* workspace, size_t workspace_bytes,
                                  ossm_stream_t stream) {
  if (!attn::valid(a)) return OSSM_EINVAL;
  if (!workspace || workspace_bytes < ossm_attn_workspace_bytes(a) || (uintptr_t)workspace % 256)
    return OSSM_EWORKSPACE;
  if (a->total_q == 0) return OSSM_OK;
  const attn::Params p{a->B, a->H, a->H_kv, a->head_dim, (int)a->total_q, (int)a->total_k, a->q, a->k, a->v, a->out,
                       a->q_stride_t, a->q_stride_h, a->k_stride_t, a->k_stride_h, a->v_stride_t, a->v_stride_h,
                       a->out_stride_t, a->out_stride_h, a->cu_q, a->cu_k, a->kv_len, a->window, a->scale};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((a->total_q + 3) / 4), a->H);
  if (a->dtype == OSSM_BF16)
    attn::attn_rows_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(p);
  else
    attn::attn_rows_kernel<__half><<<grid, 128, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}
