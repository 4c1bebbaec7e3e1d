// The next token of each row from given random numbers (ossm_sample_tokens).
//
// Every filter keeps a prefix of the candidates ordered by (logit descending,
// index ascending), so what stays is described by one 64-bit key: the logit's
// order-preserving bits above the inverted index.  One CTA per row finds the
// top-k key and then the top-p key by a radix search of 8 bits a pass (counts,
// or probability masses summed as 64-bit fixed point, whose sum does not
// depend on the order of the additions), and a last pass takes the largest
// score among the candidates at or above it.
#include <cuda_fp16.h>

#include <cmath>

#include "orthossm_b200.h"
#include "ossm_common.cuh"

namespace ossm {
namespace smp {

constexpr int kThreads = 1024;
typedef unsigned long long u64;

struct Params {
  int V;
  const void* logits;
  long long lst;
  const float* noise;
  long long nst;
  float inv_t, top_p, min_p;
  int top_k;
  const float *t_row, *p_row, *m_row;
  const int* k_row;
  int64_t* out;
};

OSSM_DEV float to_f(float v) { return v; }
OSSM_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
OSSM_DEV float to_f(__half v) { return __half2float(v); }

// A NaN or -inf logit is no candidate.
OSSM_DEV bool live(float l) { return l > -INFINITY; }

// Larger key: earlier candidate.  -0 and +0 are the same logit.
OSSM_DEV uint32_t ord(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
OSSM_DEV u64 key_of(float l, int i) { return ((u64)ord(l) << 32) | (0xffffffffu - (uint32_t)i); }
OSSM_DEV float logit_of(u64 key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// Probability relative to the first candidate (logit m): 1 at l == m, also
// where both are +inf.
OSSM_DEV float weight(float l, float m, float inv_t) {
  return l == m ? 1.f : expf(__fmul_rn(__fsub_rn(l, m), inv_t));
}
// 2^-40 steps: a row's sum stays below 2^63 for V < 2^23 equal candidates.
OSSM_DEV u64 mass_of(float w) { return (u64)__float2ull_rn(w * 0x1p40f); }

// The product and the difference are rounded one after the other (no fused
// multiply-add), so that a caller can recompute a score exactly.  A NaN (from
// NaN noise) ranks last.
OSSM_DEV float score_of(float l, float inv_t, float e) {
  const float s = __fsub_rn(__fmul_rn(l, inv_t), logf(e));
  return s == s ? s : -INFINITY;
}

struct Best {
  float s;
  int i;
};
OSSM_DEV void better(Best& a, float s, int i) {
  if (i >= 0 && (a.i < 0 || s > a.s || (s == a.s && i < a.i))) {
    a.s = s;
    a.i = i;
  }
}

OSSM_DEV u64 block_max(u64 v, u64* red) {
  for (int w = 16; w; w >>= 1) v = max(v, __shfl_xor_sync(~0u, v, w));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
  for (int w = 16; w; w >>= 1) v = max(v, __shfl_xor_sync(~0u, v, w));
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  __shared__ u64 hist[256];
  __shared__ u64 red[32];
  __shared__ u64 sh_prefix, sh_left;
  __shared__ Best bests[32];
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* lg = static_cast<const T*>(p.logits) + row * p.lst;
  const float* nz = p.noise ? p.noise + row * p.nst : nullptr;
  float inv_t = p.inv_t;
  if (p.t_row) inv_t = 1.0f / p.t_row[row];
  const bool greedy = !nz || !(inv_t > 0.f) || inv_t == INFINITY;
  const int top_k = p.k_row ? p.k_row[row] : p.top_k;
  const float top_p = p.p_row ? p.p_row[row] : p.top_p, min_p = p.m_row ? p.m_row[row] : p.min_p;

  u64 best = 0;
  for (int i = tid; i < p.V; i += kThreads) {
    const float l = to_f(lg[i]);
    if (live(l)) best = max(best, key_of(l, i));
  }
  best = block_max(best, red);
  if (best == 0 || greedy) {
    if (tid == 0) p.out[row] = best == 0 ? -1 : (int64_t)(0xffffffffu - (uint32_t)best);
    return;
  }
  const float m = logit_of(best);

  // keep = the smallest key that stays
  u64 keep = 0;
  for (int what = 0; what < 2; ++what) {  // 0: by count, 1: by mass
    u64 target;
    if (what == 0) {
      if (top_k <= 0 || top_k >= p.V) continue;
      target = top_k;
    } else {
      if (top_p >= 1.f) continue;
      u64 z = 0;
      for (int i = tid; i < p.V; i += kThreads) {
        const float l = to_f(lg[i]);
        if (live(l) && key_of(l, i) >= keep) z += mass_of(weight(l, m, inv_t));
      }
      for (int w = 16; w; w >>= 1) z += __shfl_xor_sync(~0u, z, w);
      __syncthreads();
      if ((tid & 31) == 0) red[tid >> 5] = z;
      __syncthreads();
      z = red[tid & 31];
      for (int w = 16; w; w >>= 1) z += __shfl_xor_sync(~0u, z, w);
      target = max((u64)1, (u64)__double2ull_ru((double)fmaxf(top_p, 0.f) * (double)z));
    }
    u64 prefix = 0;
    bool found = true;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < p.V; i += kThreads) {
        const float l = to_f(lg[i]);
        if (!live(l)) continue;
        const u64 key = key_of(l, i);
        if (key < keep || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
        atomicAdd(&hist[(key >> shift) & 255], what ? mass_of(weight(l, m, inv_t)) : (u64)1);
      }
      __syncthreads();
      if (tid == 0) {
        u64 left = target;
        int d = 255;
        for (; d > 0 && hist[d] < left; --d) left -= hist[d];
        sh_left = hist[d] < left ? 0 : left;  // 0: fewer than asked for are there
        sh_prefix = (prefix << 8) | d;
      }
      __syncthreads();
      target = sh_left;
      prefix = sh_prefix;
      if (target == 0) {
        found = false;
        break;
      }
    }
    if (found) keep = prefix;
  }

  Best b{0.f, -1};
  for (int i = tid; i < p.V; i += kThreads) {
    const float l = to_f(lg[i]);
    if (!live(l) || key_of(l, i) < keep) continue;
    if (min_p > 0.f && i != (int)(0xffffffffu - (uint32_t)best) && weight(l, m, inv_t) < min_p) continue;
    better(b, score_of(l, inv_t, nz[i]), i);
  }
  for (int w = 16; w; w >>= 1) better(b, __shfl_xor_sync(~0u, b.s, w), __shfl_xor_sync(~0u, b.i, w));
  if ((tid & 31) == 0) bests[tid >> 5] = b;
  __syncthreads();
  if (tid < 32) {
    b = bests[tid];
    for (int w = 16; w; w >>= 1) better(b, __shfl_xor_sync(~0u, b.s, w), __shfl_xor_sync(~0u, b.i, w));
    if (tid == 0) p.out[row] = b.i;
  }
}

}  // namespace smp
}  // namespace ossm

using namespace ossm;

extern "C" int ossm_sample_tokens(const ossm_sample_args* a, ossm_stream_t stream) {
  if (!a || a->B < 0 || a->V < 1 || a->V >= (1 << 23) || !a->logits || !a->out) return OSSM_EINVAL;
  const int el = a->dtype == OSSM_F32 ? 4 : 2;
  if ((a->dtype != OSSM_F32 && a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) || (uintptr_t)a->logits % el ||
      (uintptr_t)a->noise % 4 || (uintptr_t)a->out % 8)
    return OSSM_EINVAL;
  if (!(a->top_p >= 0.f) || !(a->min_p >= 0.f) || a->top_k < 0 || !(a->inv_temperature >= 0.f)) return OSSM_EINVAL;
  if (a->B == 0) return OSSM_OK;
  const smp::Params p{a->V, a->logits, a->logits_stride, a->noise, a->noise_stride, a->inv_temperature, a->top_p,
                      a->min_p, a->top_k, a->temperature_row, a->top_p_row, a->min_p_row, a->top_k_row, a->out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == OSSM_F32)
    smp::sample_kernel<float><<<a->B, smp::kThreads, 0, st>>>(p);
  else if (a->dtype == OSSM_BF16)
    smp::sample_kernel<__nv_bfloat16><<<a->B, smp::kThreads, 0, st>>>(p);
  else
    smp::sample_kernel<__half><<<a->B, smp::kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}
