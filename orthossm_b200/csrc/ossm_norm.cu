// A block's residual with the norms on its two sides:
//
//   n = post_norm(y),  r = x + scale gate n,  h = norm(r)
//
// norm: RMSNorm (v w / sqrt(mean v^2 + eps)) or LayerNorm (the same of v less
// its mean, plus a bias).  One pass over the rows forward, one backward; the
// gradients of what all rows share are added up in registers, a block's rows in
// order, and the blocks' sums in order by a second kernel.
//
// h is of the fp32 r, not of the rounded one that is returned.  Backward reads
// r as it was rounded where n is y itself (no norm or gate of the block's
// output): one tensor less to read; its rounding moves the normed values by
// half a step of the stream's type, as much as rounding a gradient does.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "ossm_attn.cuh"

namespace ossm {
int device_sms();
namespace nrm {

using attn::pack2;
using attn::to_f2;
typedef long long i64;

// ---------------------------------------------------------------- rows in registers
OSSM_DEV float get1(const float* p) { return *p; }
OSSM_DEV float get1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
OSSM_DEV float get1(const __half* p) { return __half2float(*p); }
OSSM_DEV void put1(float* p, float v) { *p = v; }
OSSM_DEV void put1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
OSSM_DEV void put1(__half* p, float v) { *p = __float2half_rn(v); }

// A thread's 8 N channels of a row that R threads share: N runs of eight, or,
// where a row does not start on 16 bytes or is no whole number of runs, every
// R-th channel.
template <int N>
struct Own {
  int R, t, d;
  bool vec;
  OSSM_DEV int at(int i) const { return vec ? ((i >> 3) * R + t) * 8 + (i & 7) : i * R + t; }
  OSSM_DEV bool has(int i) const { return at(i) < d; }
};
template <typename T>
OSSM_DEV void vec8(const T* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = to_f2<T>(u.x), b = to_f2<T>(u.y), c = to_f2<T>(u.z), d = to_f2<T>(u.w);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
template <>
OSSM_DEV void vec8<float>(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
OSSM_DEV void put8(T* p, const float* v) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <>
OSSM_DEV void put8<float>(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T, int N>
OSSM_DEV void load(const Own<N>& o, const T* row, float (&v)[8 * N]) {  // 0 past the row's end
  if (o.vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (o.has(8 * i)) {
        vec8<T>(row + o.at(8 * i), v + 8 * i);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[8 * i + k] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? get1(row + o.at(i)) : 0.f;
  }
}
template <typename T, int N>
OSSM_DEV void store(const Own<N>& o, T* row, const float (&v)[8 * N]) {
  if (o.vec) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (o.has(8 * i)) put8<T>(row + o.at(8 * i), v + 8 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i)
      if (o.has(i)) put1(row + o.at(i), v[i]);
  }
}
// A vector of parameters, of any of the three types; `none` where there is none.
struct Param {
  const void* p;
  int dtype;
  OSSM_DEV float one(i64 i) const {
    return dtype == OSSM_F32    ? get1(static_cast<const float*>(p) + i)
           : dtype == OSSM_BF16 ? get1(static_cast<const __nv_bfloat16*>(p) + i)
                                : get1(static_cast<const __half*>(p) + i);
  }
};
template <int N>
OSSM_DEV void load(const Own<N>& o, const Param& q, i64 from, bool vec, float none, float (&v)[8 * N]) {
  if (!q.p) {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = none;
  } else if (o.vec && !vec) {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? q.one(from + o.at(i)) : 0.f;
  } else if (q.dtype == OSSM_F32) {
    load<float>(o, static_cast<const float*>(q.p) + from, v);
  } else if (q.dtype == OSSM_BF16) {
    load<__nv_bfloat16>(o, static_cast<const __nv_bfloat16*>(q.p) + from, v);
  } else {
    load<__half>(o, static_cast<const __half*>(q.p) + from, v);
  }
}

enum { G_NONE, G_CHANNEL, G_TOKEN, G_FULL };
enum { N_NONE, N_RMS, N_LAYER };

struct Params {
  i64 T;
  int d, R;       // R threads a row
  bool vec;       // every row starts on 16 bytes and is whole runs of eight channels
  const void *x, *y;
  i64 xst, yst;
  int gate_kind;
  Param gate;
  i64 gst;
  float scale;
  int post, norm;
  Param pw, pb, w, b;
  bool gate_vec, pw_vec, pb_vec, w_vec, b_vec;  // these start on 16 bytes
  float post_eps, eps, inv_d;
  void *r, *h;
  float* stats;   // [4][T] mean and inverse deviation of r, of y
  // backward
  const void *dr, *dh;  // or NULL
  i64 drst, dhst;
  void *dx, *dy, *dgate;  // or NULL; dgate: of token and full gates
  int dgate_dtype;
  float* part;    // [blocks][sums][d]
};

// Sums over the threads of a row, the same in all of them.
template <int K>
OSSM_DEV void row_sum(float (&v)[K], int R, float (*warps)[K]) {
#pragma unroll
  for (int w = 16; w; w >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(~0u, v[k], w);
  if (R == 32) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) warps[threadIdx.x >> 5][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int i = 0; i < R / 32; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += warps[i][k];
}

// Mean and inverse deviation of a row; v becomes the normed values.
template <int N>
OSSM_DEV void normalise(const Own<N>& o, float (&v)[8 * N], int kind, float eps, float inv_d, float& mean, float& inv,
                        float (*warps)[2]) {
  mean = 0.f;
  if (kind == N_LAYER) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) s[0] += v[i];
    row_sum<2>(s, o.R, warps);
    mean = s[0] * inv_d;
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? v[i] - mean : 0.f;
  }
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8 * N; ++i) s[0] = fmaf(v[i], v[i], s[0]);
  row_sum<2>(s, o.R, warps);
  inv = 1.f / sqrtf(fmaf(s[0], inv_d, eps));
#pragma unroll
  for (int i = 0; i < 8 * N; ++i) v[i] *= inv;
}

constexpr int kWarpRows = 8;  // rows of a block where a warp takes one

// ---------------------------------------------------------------- forward
// MAXT: the most threads of a block; a block is one row, or 8 rows of a warp each.
template <typename TX, typename TY, int N, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(const __grid_constant__ Params p) {
  __shared__ float warps[MAXT / 32][2];
  const int per = blockDim.x / p.R;
  const i64 t = (i64)blockIdx.x * per + threadIdx.x / p.R;
  if (t >= p.T) return;
  const Own<N> o{p.R, (int)(threadIdx.x % p.R), p.d, p.vec};
  float v[8 * N], u[8 * N];
  load<TX>(o, static_cast<const TX*>(p.x) + t * p.xst, v);
  float mean, inv, pmean = 0.f, pinv = 1.f;
  if (p.y) {
    load<TY>(o, static_cast<const TY*>(p.y) + t * p.yst, u);
    if (p.post) {
      normalise(o, u, p.post, p.post_eps, p.inv_d, pmean, pinv, warps);
      float a[8 * N];
      load(o, p.pw, 0, p.pw_vec, 1.f, a);
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) u[i] *= a[i];
      if (p.pb.p) {
        load(o, p.pb, 0, p.pb_vec, 0.f, a);
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) u[i] += a[i];
      }
    }
    if (p.gate_kind == G_TOKEN) {
      const float g = p.gate.one(t);
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) u[i] *= g;
    } else if (p.gate_kind) {
      float a[8 * N];
      load(o, p.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, a);
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) u[i] *= a[i];
    }
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = fmaf(p.scale, u[i], v[i]);
    if (p.r) store<TX>(o, static_cast<TX*>(p.r) + t * p.d, v);
  }
  normalise(o, v, p.norm, p.eps, p.inv_d, mean, inv, warps);
  load(o, p.w, 0, p.w_vec, 1.f, u);
#pragma unroll
  for (int i = 0; i < 8 * N; ++i) v[i] *= u[i];
  if (p.b.p) {
    load(o, p.b, 0, p.b_vec, 0.f, u);
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] += u[i];
  }
  store<TY>(o, static_cast<TY*>(p.h) + t * p.d, v);
  if (p.stats && o.t == 0) {
    p.stats[t] = mean;
    p.stats[p.T + t] = inv;
    if (p.post) {
      p.stats[2 * p.T + t] = pmean;
      p.stats[3 * p.T + t] = pinv;
    }
  }
}

// ---------------------------------------------------------------- backward
enum { S_W, S_B, S_GATE, S_PW, S_PB, kSums };  // sums over the rows

// FULL: the block's output has a norm or a gate, so y is read.
template <typename TX, typename TY, int N, bool FULL, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kHere = FULL ? (int)kSums : 2;
  __shared__ float warps[MAXT / 32][2];
  extern __shared__ float smem[];  // to join the sums of a block's rows
  const int per = blockDim.x / p.R, mine = threadIdx.x / p.R;
  const Own<N> o{p.R, (int)(threadIdx.x % p.R), p.d, p.vec};
  float sum[kHere][8 * N];
#pragma unroll
  for (int k = 0; k < kHere; ++k)
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) sum[k][i] = 0.f;
  for (i64 t = (i64)blockIdx.x * per + mine; t < p.T; t += (i64)gridDim.x * per) {
    float v[8 * N], g[8 * N], n[8 * N], a[8 * N];  // normed r; gradient of r; block's output
    const float inv = p.stats[p.T + t], mean = p.norm == N_LAYER ? p.stats[t] : 0.f;
    if (FULL) {
      load<TX>(o, static_cast<const TX*>(p.x) + t * p.xst, v);
      load<TY>(o, static_cast<const TY*>(p.y) + t * p.yst, n);
    } else {
      load<TX>(o, static_cast<const TX*>(p.r) + t * p.xst, v);
    }
    float pinv = 1.f, pmean = 0.f, gt = 1.f;
    if (FULL) {
      if (p.post) {
        pinv = p.stats[3 * p.T + t];
        if (p.post == N_LAYER) pmean = p.stats[2 * p.T + t];
      }
      if (p.gate_kind == G_TOKEN) gt = p.gate.one(t);
      // r again: x + scale gate (pv pw + pb)
      float c[8 * N];
      load(o, p.pw, 0, p.pw_vec, 1.f, a);
      if (p.gate_kind == G_CHANNEL || p.gate_kind == G_FULL)
        load(o, p.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, c);
      else
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) c[i] = gt;
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) a[i] *= (n[i] - pmean) * pinv;
      if (p.pb.p) {
        load(o, p.pb, 0, p.pb_vec, 0.f, g);
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) a[i] += g[i];
      }
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) v[i] = fmaf(p.scale, c[i] * a[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? (v[i] - mean) * inv : 0.f;
    if (p.dr)
      load<TX>(o, static_cast<const TX*>(p.dr) + t * p.drst, g);
    else
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) g[i] = 0.f;
    if (p.dh) {
      float e[8 * N], f[8 * N];
      load<TY>(o, static_cast<const TY*>(p.dh) + t * p.dhst, e);
      load(o, p.w, 0, p.w_vec, 1.f, f);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) {
        sum[S_W][i] = fmaf(e[i], v[i], sum[S_W][i]);
        sum[S_B][i] += e[i];
        e[i] *= f[i];
        s[0] = fmaf(e[i], v[i], s[0]);
        s[1] += e[i];
      }
      row_sum<2>(s, p.R, warps);
      const float m0 = s[0] * p.inv_d, m1 = p.norm == N_LAYER ? s[1] * p.inv_d : 0.f;
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) g[i] = fmaf(inv, e[i] - m1 - v[i] * m0, g[i]);
    }
    if (p.dx) store<TX>(o, static_cast<TX*>(p.dx) + t * p.d, g);
    if (!FULL) {
      if (p.dy) {
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) g[i] *= p.scale;
        store<TY>(o, static_cast<TY*>(p.dy) + t * p.d, g);
      }
      continue;
    }
    if (FULL) {
      // a: the block's output after its norm; g: the gradient of r
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) {
        g[i] *= p.scale;
        a[i] = o.has(i) ? a[i] * g[i] : 0.f;  // the gate's gradient
        s[0] += a[i];
        sum[S_GATE][i] += a[i];
      }
      if (p.gate_kind == G_TOKEN) {
        if (p.dgate) {
          row_sum<2>(s, p.R, warps);
          if (o.t == 0) {
            if (p.dgate_dtype == OSSM_F32) put1(static_cast<float*>(p.dgate) + t, s[0]);
            else if (p.dgate_dtype == OSSM_BF16) put1(static_cast<__nv_bfloat16*>(p.dgate) + t, s[0]);
            else put1(static_cast<__half*>(p.dgate) + t, s[0]);
          }
        }
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) g[i] *= gt;
      } else if (p.gate_kind) {
        if (p.gate_kind == G_FULL && p.dgate) {
          if (p.dgate_dtype == OSSM_F32) store<float>(o, static_cast<float*>(p.dgate) + t * p.d, a);
          else if (p.dgate_dtype == OSSM_BF16) store<__nv_bfloat16>(o, static_cast<__nv_bfloat16*>(p.dgate) + t * p.d, a);
          else store<__half>(o, static_cast<__half*>(p.dgate) + t * p.d, a);
        }
        float c[8 * N];
        load(o, p.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, c);
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) g[i] *= c[i];
      }
      if (p.post) {
        load(o, p.pw, 0, p.pw_vec, 1.f, a);
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) {
          n[i] = o.has(i) ? (n[i] - pmean) * pinv : 0.f;
          sum[S_PW][i] = fmaf(g[i], n[i], sum[S_PW][i]);
          sum[S_PB][i] += g[i];
          g[i] = o.has(i) ? g[i] * a[i] : 0.f;
          s[0] = fmaf(g[i], n[i], s[0]);
          s[1] += g[i];
        }
        row_sum<2>(s, p.R, warps);
        const float m0 = s[0] * p.inv_d, m1 = p.post == N_LAYER ? s[1] * p.inv_d : 0.f;
#pragma unroll
        for (int i = 0; i < 8 * N; ++i) g[i] = pinv * (g[i] - m1 - n[i] * m0);
      }
      if (p.dy) store<TY>(o, static_cast<TY*>(p.dy) + t * p.d, g);
    }
  }
  if (!p.part) return;
  // the block's sums, its rows' threads in order
#pragma unroll
  for (int k = 0; k < kHere; ++k) {
    float* to = p.part + ((i64)blockIdx.x * kHere + k) * p.d;
    if (per == 1) {
#pragma unroll
      for (int i = 0; i < 8 * N; ++i)
        if (o.has(i)) to[o.at(i)] = sum[k][i];
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) smem[(mine * 8 * N + i) * p.R + o.t] = sum[k][i];
    __syncthreads();
    for (int i = mine; i < 8 * N; i += per) {
      float all = 0.f;
      for (int q = 0; q < per; ++q) all += smem[(q * 8 * N + i) * p.R + o.t];
      if (o.has(i)) to[o.at(i)] = all;
    }
  }
}

struct Outs {
  void* to[kSums];
  int dtype[kSums];
};
// Adds the blocks' sums up in order: 32 channels a block, 8 runs of blocks side by side.
__global__ void __launch_bounds__(256) norm_sums_kernel(const float* part, int blocks, int sums, int d, const __grid_constant__ Outs outs) {
  __shared__ float s[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5, k = blockIdx.y;
  if (!outs.to[k]) return;
  const int each = (blocks + 7) / 8;
  float a = 0.f;
  if (c < d)
#pragma unroll 8
    for (int b = run * each; b < min(blocks, (run + 1) * each); ++b) a += __ldg(part + ((i64)b * sums + k) * d + c);
  s[run][threadIdx.x & 31] = a;
  __syncthreads();
  if (run || c >= d) return;
  for (int i = 1; i < 8; ++i) a += s[i][threadIdx.x];
  if (outs.dtype[k] == OSSM_F32) put1(static_cast<float*>(outs.to[k]) + c, a);
  else if (outs.dtype[k] == OSSM_BF16) put1(static_cast<__nv_bfloat16*>(outs.to[k]) + c, a);
  else put1(static_cast<__half*>(outs.to[k]) + c, a);
}

// ---------------------------------------------------------------- host
bool float_type(int t) { return t == OSSM_F32 || t == OSSM_BF16 || t == OSSM_F16; }
size_t size_of(int t) { return t == OSSM_F32 ? 4 : 2; }

bool valid(const ossm_norm_args* a, bool bwd) {
  if (!a || a->tokens < 0 || a->tokens > (1LL << 31) - 1 || a->dim < 1 || a->dim > 16384) return false;
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
  if (full ? (!a->x || a->x_stride < a->dim || !a->y || a->y_stride < a->dim) : (!a->r || a->x_stride < a->dim)) return false;
  if ((a->grad_r && a->grad_r_stride < a->dim) || (a->grad_h && a->grad_h_stride < a->dim)) return false;
  return a->grad_r || a->grad_h;
}

struct Plan {
  int R, N, per, blocks, sums;
  bool full;
  size_t bytes;
};
// Threads of a row: a warp up to 512 channels, then as many as make 16 channels each.
Plan plan_of(const ossm_norm_args* a, bool bwd) {
  Plan q{};
  q.full = a->post_norm || a->gate_kind;
  const int runs = (a->dim + 7) / 8;
  q.N = runs <= 32 ? 1 : 2;
  q.R = runs <= 64 ? 32 : (runs + 63) / 64 * 32;
  q.per = q.R == 32 ? kWarpRows : 1;
  const i64 rows = std::max<i64>(1, (a->tokens + q.per - 1) / q.per);
  q.sums = q.full ? (int)kSums : 2;
  if (bwd) {
    q.blocks = (int)std::min<i64>(rows, 4LL * device_sms());
    q.bytes = (size_t)q.blocks * q.sums * a->dim * 4;
  }
  return q;
}

Params params_of(const ossm_norm_args* a, const Plan& q, bool bwd) {
  Params p{};
  const size_t sx = size_of(a->stream_dtype), sy = size_of(a->dtype);
  bool vec = a->dim % 8 == 0;
  auto rows = [&](const void* ptr, i64 st, size_t sz) {
    if (ptr && ((uintptr_t)ptr % 16 || st * sz % 16)) vec = false;
  };
  rows(a->x, a->x_stride, sx);
  rows(a->y, a->y_stride, sy);
  rows(a->r, bwd && !q.full ? a->x_stride : a->dim, sx);
  if (bwd) {
    rows(a->grad_r, a->grad_r_stride, sx);
    rows(a->grad_h, a->grad_h_stride, sy);
    rows(a->grad_x, a->dim, sx);
    rows(a->grad_y, a->dim, sy);
    if (a->gate_kind == OSSM_GATE_FULL) rows(a->grad_gate, a->dim, size_of(a->gate_dtype));
  } else {
    rows(a->h, a->dim, sy);
  }
  p.T = a->tokens, p.d = a->dim, p.R = q.R, p.vec = vec;
  p.x = a->x, p.y = a->y, p.xst = a->x_stride, p.yst = a->y_stride;
  p.gate_kind = a->gate_kind, p.gate = {a->gate, a->gate_dtype}, p.gst = a->gate_stride;
  p.scale = a->scale, p.post = a->post_norm, p.norm = a->norm;
  p.w = {a->weight, a->weight_dtype}, p.b = {a->bias, a->bias_dtype};
  p.pw = {a->post_weight, a->post_weight_dtype}, p.pb = {a->post_bias, a->post_bias_dtype};
  auto aligned = [](const void* ptr) { return (uintptr_t)ptr % 16 == 0; };
  p.gate_vec = aligned(a->gate) && (a->gate_kind != OSSM_GATE_FULL || a->gate_stride * size_of(a->gate_dtype) % 16 == 0);
  p.w_vec = aligned(a->weight), p.b_vec = aligned(a->bias);
  p.pw_vec = aligned(a->post_weight), p.pb_vec = aligned(a->post_bias);
  p.post_eps = a->post_eps, p.eps = a->eps, p.inv_d = 1.f / a->dim;
  p.r = a->r, p.h = a->h, p.stats = a->stats;
  p.dr = a->grad_r, p.dh = a->grad_h, p.drst = a->grad_r_stride, p.dhst = a->grad_h_stride;
  p.dx = a->grad_x, p.dy = a->grad_y, p.dgate = a->grad_gate, p.dgate_dtype = a->gate_dtype;
  return p;
}

template <typename TX, typename TY>
int forward(const ossm_norm_args* a, cudaStream_t st) {
  const Plan q = plan_of(a, false);
  const Params p = params_of(a, q, false);
  const unsigned grid = (unsigned)((a->tokens + q.per - 1) / q.per);
  auto kern = q.N == 1     ? norm_fwd_kernel<TX, TY, 1, 256>
              : q.R <= 256 ? norm_fwd_kernel<TX, TY, 2, 256>
                           : norm_fwd_kernel<TX, TY, 2, 1024>;
  kern<<<grid, q.R * q.per, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

template <typename TX, typename TY>
int backward(const ossm_norm_args* a, const Plan& q, float* part, cudaStream_t st) {
  Params p = params_of(a, q, true);
  const bool sums = a->grad_weight || a->grad_bias || a->grad_post_weight || a->grad_post_bias ||
                    (a->gate_kind == OSSM_GATE_CHANNEL && a->grad_gate);
  p.part = sums ? part : nullptr;
  if (a->gate_kind == OSSM_GATE_CHANNEL) p.dgate = nullptr;
  const bool big = q.R > 256;
  auto kern = q.full ? (q.N == 1 ? norm_bwd_kernel<TX, TY, 1, true, 256>
                        : big    ? norm_bwd_kernel<TX, TY, 2, true, 1024>
                                 : norm_bwd_kernel<TX, TY, 2, true, 256>)
                     : (q.N == 1 ? norm_bwd_kernel<TX, TY, 1, false, 256>
                        : big    ? norm_bwd_kernel<TX, TY, 2, false, 1024>
                                 : norm_bwd_kernel<TX, TY, 2, false, 256>);
  const size_t smem = q.per > 1 ? (size_t)q.per * 8 * q.N * q.R * 4 : 0;
  kern<<<q.blocks, q.R * q.per, smem, st>>>(p);
  if (sums) {
    Outs o{};
    o.to[S_W] = a->grad_weight, o.dtype[S_W] = a->weight_dtype;
    o.to[S_B] = a->grad_bias, o.dtype[S_B] = a->bias_dtype;
    if (a->gate_kind == OSSM_GATE_CHANNEL) o.to[S_GATE] = a->grad_gate, o.dtype[S_GATE] = a->gate_dtype;
    o.to[S_PW] = a->grad_post_weight, o.dtype[S_PW] = a->post_weight_dtype;
    o.to[S_PB] = a->grad_post_bias, o.dtype[S_PB] = a->post_bias_dtype;
    norm_sums_kernel<<<dim3((a->dim + 31) / 32, q.sums), 256, 0, st>>>(part, q.blocks, q.sums, a->dim, o);
  }
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

template <typename F>
int by_type(const ossm_norm_args* a, F f) {
  typedef __nv_bfloat16 bf;
  typedef __half hf;
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
