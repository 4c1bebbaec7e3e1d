// A block's residual with the norms on its two sides:
//
//   n = post_norm(y),  r = x + scale gate n,  h = norm(r)
//
// norm: RMSNorm (v w / sqrt(mean v^2 + eps)) or LayerNorm (the same of v less
// its mean, plus a bias).  One pass over the rows forward, one backward; the
// gradients of what all rows share are added up in registers, a block's rows in
// order, and the blocks' sums in order by a second kernel.
//
// h is of the fp32 r, not of the rounded one that is returned, and so are the
// gradients: backward adds x and y again, unless r is fp32 itself.  Normed values
// of a rounded r are off by half a step each, and the gradients are differences
// of them: dx = inv (e - v mean(e v) - mean(e)) takes off what is parallel to v, and
// LayerNorm's v is less its mean.  (RMSNorm of 512 channels with e about parallel
// to v, dx from the rounded r: off by 1.1 times its norm, bf16 1.7e-3 from x and y.
// LayerNorm, 60364 rows of 3 channels, bf16: 0.19 and 1.6e-3.)
//
// What bounds it: HBM where there are few sums (131072 x 512 bf16, RMSNorm: 89 us
// forward, 111 backward, 6.0 TB/s each); with a norm and a gate of y the
// latency of a row, whose two sums wait for each other with two rows an SM (16384 x
// 2048, fp32 stream: 80 and 175 us, 5.0 and 3.5 TB/s).
#pragma once

#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "ossm_attn.cuh"
#include "ossm_sm100.cuh"

namespace ossm {
int device_sms();
namespace nrm {

using attn::allow_smem;
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
template <int N, bool VEC>
struct Own {
  static constexpr bool vec = VEC;
  int R, t, d;
  OSSM_DEV int at(int i) const { return VEC ? ((i >> 3) * R + t) * 8 + (i & 7) : i * R + t; }
  OSSM_DEV bool has(int i) const { return VEC ? ((i >> 3) * R + t) * 8 < d : at(i) < d; }  // whole runs of eight
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
template <typename T, int N, bool VEC>
OSSM_DEV void load(const Own<N, VEC>& o, const T* row, float (&v)[8 * N]) {  // 0 past the row's end
  if (VEC) {
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
template <typename T, int N, bool VEC>
OSSM_DEV void store(const Own<N, VEC>& o, T* row, const float (&v)[8 * N]) {
  if (VEC) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (o.has(8 * i)) put8<T>(row + o.at(8 * i), v + 8 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i)
      if (o.has(i)) put1(row + o.at(i), v[i]);
  }
}
// A vector of parameters, of any of the three types.  The kernels keep a copy in
// fp32 in shared memory where it fits beside the rows.
struct Param {
  const void* p;
  int dtype;
  const float* shared;  // a copy in shared memory, or NULL
  OSSM_DEV float one(i64 i) const {
    return dtype == OSSM_F32    ? get1(static_cast<const float*>(p) + i)
           : dtype == OSSM_BF16 ? get1(static_cast<const __nv_bfloat16*>(p) + i)
                                : get1(static_cast<const __half*>(p) + i);
  }
};
template <int N, bool VEC>
OSSM_DEV void load(const Own<N, VEC>& o, const Param& q, i64 from, bool vec, float none, float (&v)[8 * N]) {
  if (!q.p) {
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? none : 0.f;
  } else if (q.shared) {
    load<float>(o, q.shared, v);
  } else if (VEC && !vec) {
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
  int stages, stage_bytes;  // of the ring of a row's threads
  bool shared;              // parameters are copied to shared memory, behind the rows
  uint32_t* status;
};

// The rows of up to four tensors on their way to the threads that share them.
// Where rows are whole 16-byte pieces, bulk copies bring them into a ring in
// shared memory several rows ahead; otherwise they are read where they lie.
// (A row ahead in registers kept 48 KB an SM on its way and cost 24 to 48 of
// them: 131072 x 512 bf16, backward: 119 us.)
constexpr int kMaxStages = 8;
#ifndef OSSM_NORM_POLLS
#define OSSM_NORM_POLLS (1u << 22)  // of a wait for a row; a test compiles the kernels with none
#endif
struct Tensor {
  const char* p;  // NULL: not there
  i64 stride;     // in bytes
  int bytes, at;  // of a row; where in a stage
};
template <bool VEC>
struct Rows {
  Tensor t[4];
  char* ring;          // of this row's threads
  uint64_t* full;
  int stages, stage_bytes, R, lane;
  i64 step, T;
  uint32_t* status;
  uint32_t slot, turn;  // of the row at hand
  OSSM_DEV void fetch(i64 row, uint32_t to) {  // one thread
    sm100::mbar_expect_tx(full + to, stage_bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t[i].p) sm100::bulk_load(ring + to * stage_bytes + t[i].at, t[i].p + row * t[i].stride, t[i].bytes, full + to);
  }
  OSSM_DEV void begin(i64 first) {
    if (!VEC) return;
    if (lane == 0) {
      for (int i = 0; i < stages; ++i) sm100::mbar_init(full + i, 1);
      sm100::fence_mbar_init();
      for (int i = 0; i < stages && first + i * step < T; ++i) fetch(first + i * step, i);
    }
    meet();
  }
  OSSM_DEV void meet() const {
    if (R == 32) __syncwarp(); else __syncthreads();
  }
  // For the row at hand.  A thread whose wait runs out goes on without waiting;
  // the one that issues copies issues no more, and stays until those on their
  // way have landed: none may be when the ring is used again or the block ends.
  OSSM_DEV void wait(i64 row) {
    if (!VEC || turn > 1 || sm100::mbar_wait(full + slot, turn, OSSM_NORM_POLLS)) return;
    if (status) atomicExch(status, (uint32_t)OSSM_ETIMEOUT);
    if (lane == 0) {
      for (int i = 0; i < stages && row + i * step < T; ++i) {
        const bool next = (int)slot + i >= stages;
        sm100::mbar_wait(full + slot + i - (next ? stages : 0), turn ^ (next ? 1 : 0));
      }
    }
    T = 0, turn |= 2;
  }
  // Tensor i's row `row`, the row at hand.
  template <typename E, int N>
  OSSM_DEV void get(const Own<N, VEC>& o, int i, i64 row, float (&v)[8 * N]) const {
    load<E>(o, reinterpret_cast<const E*>(VEC ? ring + slot * stage_bytes + t[i].at : t[i].p + row * t[i].stride), v);
  }
  OSSM_DEV void taken(i64 row) {  // all threads have met since they got what they need of it
    if (!VEC) return;
    if (R == 32) __syncwarp();
    if (lane == 0 && row + stages * step < T) fetch(row + stages * step, slot);
    if (++slot == stages) slot = 0, turn ^= 1;
  }
};

// Arithmetic on a thread's channels, two an instruction.
OSSM_DEV float2 both(float f) { return make_float2(f, f); }
template <int M>
OSSM_DEV float2 pair(const float (&v)[M], int i) { return make_float2(v[2 * i], v[2 * i + 1]); }
template <int M>
OSSM_DEV void set(float (&v)[M], int i, float2 f) { v[2 * i] = f.x, v[2 * i + 1] = f.y; }
template <int M>
OSSM_DEV void mul(float (&a)[M], const float (&b)[M]) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(a, i, mul2(pair(a, i), pair(b, i)));
}
template <int M>
OSSM_DEV void mul(float (&a)[M], float f) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(a, i, mul2(pair(a, i), both(f)));
}
template <int M>
OSSM_DEV void add(float (&a)[M], const float (&b)[M]) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(a, i, attn::add2(pair(a, i), pair(b, i)));
}
template <int M>
OSSM_DEV void add(float (&a)[M], float f) {
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(a, i, attn::add2(pair(a, i), both(f)));
}
template <int M>
OSSM_DEV void fma(float (&d)[M], const float (&a)[M], const float (&b)[M]) {  // d += a b
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(d, i, fma2(pair(a, i), pair(b, i), pair(d, i)));
}
template <int M>
OSSM_DEV void fma(float (&d)[M], const float (&a)[M], float f) {  // d += a f
#pragma unroll
  for (int i = 0; i < M / 2; ++i) set(d, i, fma2(pair(a, i), both(f), pair(d, i)));
}
template <int M>
OSSM_DEV float dot(const float (&a)[M], const float (&b)[M]) {
  float2 s = both(0.f);
#pragma unroll
  for (int i = 0; i < M / 2; ++i) s = fma2(pair(a, i), pair(b, i), s);
  return s.x + s.y;
}
template <int M>
OSSM_DEV float total(const float (&a)[M]) {
  float2 s = both(0.f);
#pragma unroll
  for (int i = 0; i < M / 2; ++i) s = attn::add2(s, pair(a, i));
  return s.x + s.y;
}

// Sums over the threads of a row, the same in all of them.  Of two sums the
// lower lanes of a warp take one and the upper ones the other.  Rows of several
// warps take the two buffers in turn, so that one barrier a sum is enough.
template <int MAXT>
struct RowSum {
  float (*buf)[2][32];
  int R, turn;
  OSSM_DEV float warp_sum(float v) const {
#pragma unroll
    for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(~0u, v, w);
    return v;
  }
  OSSM_DEV void operator()(float& v) {
    v = warp_sum(v);
    if (R == 32) return;
    const int lane = threadIdx.x & 31;
    if (lane == 0) buf[turn][0][threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < R / 32 ? buf[turn][0][lane] : 0.f;
    constexpr int W = MAXT > 256 ? 8 : 4;  // the warps' sums lie in the first 8 or 16 lanes
#pragma unroll
    for (int w = W; w; w >>= 1) v += __shfl_xor_sync(~0u, v, w);
    v = __shfl_sync(~0u, v, 0);
    turn ^= 1;
  }
  OSSM_DEV void operator()(float& a, float& b) {
    const int lane = threadIdx.x & 31;
    const bool upper = lane & 16;
    float v = upper ? b : a;
    v += __shfl_xor_sync(~0u, upper ? a : b, 16);
#pragma unroll
    for (int w = 8; w; w >>= 1) v += __shfl_xor_sync(~0u, v, w);
    if (R > 32) {
      if ((lane & 15) == 0) buf[turn][lane >> 4][threadIdx.x >> 5] = v;
      __syncthreads();
      v = (lane & 15) < R / 32 ? buf[turn][lane >> 4][lane & 15] : 0.f;  // of up to 16 warps
#pragma unroll
      for (int w = MAXT > 256 ? 8 : 4; w; w >>= 1) v += __shfl_xor_sync(~0u, v, w);
      turn ^= 1;
    }
    a = __shfl_sync(~0u, v, 0), b = __shfl_sync(~0u, v, 16);
  }
};

// Mean and inverse deviation of a row; v becomes the normed values.
template <int MAXT, int N, bool VEC>
OSSM_DEV void normalise(const Own<N, VEC>& o, float (&v)[8 * N], int kind, float eps, float inv_d, float& mean, float& inv,
                        RowSum<MAXT>& sum) {
  mean = 0.f;
  if (kind == N_LAYER) {
    mean = total(v);
    sum(mean);
    mean *= inv_d;
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) v[i] = o.has(i) ? v[i] - mean : 0.f;
  }
  float s = dot(v, v);
  sum(s);
  inv = 1.f / sqrtf(fmaf(s, inv_d, eps));
  mul(v, inv);
}

constexpr int kWarpRows = 8;  // rows of a block where a warp takes one

// The parameters that all rows share, copied to shared memory.
struct Shares {
  Param w, b, pw, pb, gate;
  OSSM_DEV Shares(const Params& p, char* ring, int per) : w(p.w), b(p.b), pw(p.pw), pb(p.pb), gate(p.gate) {
    if (!p.shared) return;
    float* to = reinterpret_cast<float*>(ring + (i64)per * p.stages * p.stage_bytes);
    auto copy = [&](Param& q) {
      if (!q.p) return;
      for (int i = threadIdx.x; i < p.d; i += blockDim.x) to[i] = q.one(i);
      q.shared = to;
      to += p.d;
    };
    copy(w), copy(b), copy(pw), copy(pb);
    if (p.gate_kind == G_CHANNEL) copy(gate);
    __syncthreads();
  }
};

// ---------------------------------------------------------------- forward
// MAXT: the most threads of a block; a block is one row, or 8 rows of a warp each.
template <typename TX, typename TY, int N, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= 256 ? 3 : 1) norm_fwd_kernel(const __grid_constant__ Params p) {
  __shared__ float buf[2][2][32];
  __shared__ uint64_t full[kWarpRows][kMaxStages];
  extern __shared__ __align__(16) char ring[];
  RowSum<MAXT> sum{buf, p.R, 0};
  const int per = blockDim.x / p.R, mine = threadIdx.x / p.R;
  const i64 step = (i64)gridDim.x * per;
  i64 t = (i64)blockIdx.x * per + mine;
  const Own<N, VEC> o{p.R, (int)(threadIdx.x % p.R), p.d};
  constexpr int SX = sizeof(TX), SY = sizeof(TY);
  Rows<VEC> rows{{{static_cast<const char*>(p.x), p.xst * SX, p.d * SX, 0},
                  {static_cast<const char*>(p.y), p.yst * SY, p.d * SY, p.d * SX}},
                 ring + mine * p.stages * p.stage_bytes, full[mine], p.stages, p.stage_bytes, p.R, o.t, step, p.T,
                 p.status, 0, 0};
  rows.begin(t);
  const Shares own(p, ring, per);
  for (; t < p.T; t += step) {
    float v[8 * N], u[8 * N];
    rows.wait(t);
    rows.template get<TX>(o, 0, t, v);
    if (p.y) rows.template get<TY>(o, 1, t, u);
    float mean, inv, pmean = 0.f, pinv = 1.f;
    if (p.y) {
      if (p.post) {
        normalise(o, u, p.post, p.post_eps, p.inv_d, pmean, pinv, sum);
        float a[8 * N];
        load(o, own.pw, 0, p.pw_vec, 1.f, a);
        mul(u, a);
        if (p.pb.p) {
          load(o, own.pb, 0, p.pb_vec, 0.f, a);
          add(u, a);
        }
      }
      if (p.gate_kind == G_TOKEN) {
        const float g = p.gate.one(t);
        mul(u, g);
      } else if (p.gate_kind) {
        float a[8 * N];
        load(o, own.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, a);
        mul(u, a);
      }
      fma(v, u, p.scale);
      store<TX>(o, static_cast<TX*>(p.r) + t * p.d, v);
    }
    normalise(o, v, p.norm, p.eps, p.inv_d, mean, inv, sum);
    rows.taken(t);
    load(o, own.w, 0, p.w_vec, 1.f, u);
    mul(v, u);
    if (p.b.p) {
      load(o, own.b, 0, p.b_vec, 0.f, u);
      add(v, u);
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
}

// ---------------------------------------------------------------- backward
enum { S_W, S_B, S_GATE, S_PW, S_PB, kSums };  // sums over the rows

// SUMS: how many of the sums are kept: the weight's, the bias's too, or all,
// where the block's output has a norm or a gate.
template <typename TX, typename TY, int N, bool VEC, int SUMS, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= 256 && (N == 1 || SUMS <= 2) ? 2 : 1)
    norm_bwd_kernel(const __grid_constant__ Params p) {
  constexpr bool FULL = SUMS == (int)kSums;
  __shared__ float buf[2][2][32];
  __shared__ uint64_t full[kWarpRows][kMaxStages];
  extern __shared__ __align__(16) char ring[];
  RowSum<MAXT> row_sum{buf, p.R, 0};
  const int per = blockDim.x / p.R, mine = threadIdx.x / p.R;
  const i64 step = (i64)gridDim.x * per;
  const Own<N, VEC> o{p.R, (int)(threadIdx.x % p.R), p.d};
  float sum[SUMS][8 * N];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) sum[k][i] = 0.f;
  i64 t = (i64)blockIdx.x * per + mine;
  constexpr int SX = sizeof(TX), SY = sizeof(TY);
  // x (or r alone), the gradient of r, of h, y
  const int at1 = p.d * SX, at2 = at1 + (p.dr ? p.d * SX : 0), at3 = at2 + (p.dh ? p.d * SY : 0);
  Rows<VEC> rows{{{static_cast<const char*>(p.y ? p.x : p.r), p.xst * SX, p.d * SX, 0},
                  {static_cast<const char*>(p.dr), p.drst * SX, p.d * SX, at1},
                  {static_cast<const char*>(p.dh), p.dhst * SY, p.d * SY, at2},
                  {static_cast<const char*>(p.y), p.yst * SY, p.d * SY, at3}},
                 ring + mine * p.stages * p.stage_bytes, full[mine], p.stages, p.stage_bytes, p.R, o.t, step, p.T,
                 p.status, 0, 0};
  rows.begin(t);
  const Shares own(p, ring, per);
  float inv_a = 0.f, mean_a = 0.f, pinv_a = 1.f, pmean_a = 0.f;  // of the next row
  auto stats = [&](i64 row) {
    if (row >= p.T) return;
    inv_a = __ldg(p.stats + p.T + row);
    if (p.norm == N_LAYER) mean_a = __ldg(p.stats + row);
    if (FULL && p.post) {
      pinv_a = __ldg(p.stats + 3 * p.T + row);
      if (p.post == N_LAYER) pmean_a = __ldg(p.stats + 2 * p.T + row);
    }
  };
  stats(t);
  for (; t < p.T; t += step) {
    // past the row's end e and a are 0, and nothing else of there is used
    float v[8 * N], g[8 * N], e[8 * N], n[FULL ? 8 * N : 1], a[FULL ? 8 * N : 1];
    const float inv = inv_a, mean = mean_a, pinv = pinv_a, pmean = pmean_a;
    stats(t + step);
    rows.wait(t);
    rows.template get<TX>(o, 0, t, v);
    if (p.dr) {
      rows.template get<TX>(o, 1, t, g);
    } else {
#pragma unroll
      for (int i = 0; i < 8 * N; ++i) g[i] = 0.f;
    }
    if (p.dh) rows.template get<TY>(o, 2, t, e);
    if constexpr (FULL) {
      rows.template get<TY>(o, 3, t, n);
    } else if (p.y) {
      float u[8 * N];
      rows.template get<TY>(o, 3, t, u);
      fma(v, u, p.scale);
    }
    float gt = 1.f;
    if constexpr (FULL) {
      // n becomes y normed (or y); a: the block's output after that; v: r again
      if (p.post) {
        if (p.post == N_LAYER) add(n, -pmean);
        mul(n, pinv);
      }
      float c[8 * N];
      load(o, own.pw, 0, p.pw_vec, 1.f, a);
      mul(a, n);
      if (p.pb.p) {
        load(o, own.pb, 0, p.pb_vec, 0.f, c);
        add(a, c);
      }
      if (p.gate_kind == G_TOKEN) gt = p.gate.one(t);
      if (p.gate_kind == G_CHANNEL || p.gate_kind == G_FULL) {
        load(o, own.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, c);
        mul(c, a);
        fma(v, c, p.scale);
      } else {
        fma(v, a, p.scale * gt);
      }
    }
    if (p.norm == N_LAYER) add(v, -mean);
    mul(v, inv);
    if (p.dh) {
      fma(sum[S_W], e, v);
      if (SUMS > 1) add(sum[SUMS > 1 ? S_B : 0], e);
      if (own.w.p) {
        float f[8 * N];
        load(o, own.w, 0, p.w_vec, 1.f, f);
        mul(e, f);
      }
      float m0 = dot(e, v), m1 = 0.f;
      if (p.norm == N_LAYER) {
        m1 = total(e);
        row_sum(m0, m1);
        m1 *= p.inv_d;
      } else {
        row_sum(m0);
      }
      rows.taken(t);
      m0 *= p.inv_d;
      fma(e, v, -m0);
      if (p.norm == N_LAYER) add(e, -m1);
      fma(g, e, inv);
    } else {
      rows.meet();
      rows.taken(t);
    }
    if (p.dx) store<TX>(o, static_cast<TX*>(p.dx) + t * p.d, g);
    if constexpr (!FULL) {
      if (p.dy) {
        mul(g, p.scale);
        store<TY>(o, static_cast<TY*>(p.dy) + t * p.d, g);
      }
    } else {
      mul(g, p.scale);
      mul(a, g);  // the gate's gradient
      add(sum[S_GATE], a);
      if (p.gate_kind == G_TOKEN) {
        if (p.dgate) {
          float s = total(a);
          row_sum(s);
          if (o.t == 0) {
            if (p.dgate_dtype == OSSM_F32) put1(static_cast<float*>(p.dgate) + t, s);
            else if (p.dgate_dtype == OSSM_BF16) put1(static_cast<__nv_bfloat16*>(p.dgate) + t, s);
            else put1(static_cast<__half*>(p.dgate) + t, s);
          }
        }
        mul(g, gt);
      } else if (p.gate_kind) {
        if (p.gate_kind == G_FULL && p.dgate) {
          if (p.dgate_dtype == OSSM_F32) store<float>(o, static_cast<float*>(p.dgate) + t * p.d, a);
          else if (p.dgate_dtype == OSSM_BF16) store<__nv_bfloat16>(o, static_cast<__nv_bfloat16*>(p.dgate) + t * p.d, a);
          else store<__half>(o, static_cast<__half*>(p.dgate) + t * p.d, a);
        }
        load(o, own.gate, p.gate_kind == G_FULL ? t * p.gst : 0, p.gate_vec, 1.f, a);
        mul(g, a);
      }
      if (p.post) {
        fma(sum[S_PW], g, n);
        add(sum[S_PB], g);
        load(o, own.pw, 0, p.pw_vec, 1.f, a);
        mul(g, a);
        float m0 = dot(g, n), m1 = 0.f;
        if (p.post == N_LAYER) {
          m1 = total(g);
          row_sum(m0, m1);
          m1 *= p.inv_d;
        } else {
          row_sum(m0);
        }
        m0 *= p.inv_d;
        fma(g, n, -m0);
        if (p.post == N_LAYER) add(g, -m1);
        mul(g, pinv);
      }
      if (p.dy) store<TY>(o, static_cast<TY*>(p.dy) + t * p.d, g);
    }
  }
  if (!p.part) return;
  float* smem = reinterpret_cast<float*>(ring);  // the rows are through
  // the block's sums, its rows' threads in order
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
    float* to = p.part + ((i64)blockIdx.x * SUMS + k) * p.d;
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
// Adds the blocks' sums up in order: 32 channels a block, 32 runs of blocks side by side.
static __global__ void __launch_bounds__(1024)
    norm_sums_kernel(const float* part, int blocks, int sums, int d, const __grid_constant__ Outs outs) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, run = threadIdx.x >> 5, k = blockIdx.y;
  if (!outs.to[k]) return;
  const int each = (blocks + 31) / 32;
  float a = 0.f;
  if (c < d)
#pragma unroll 8
    for (int b = run * each; b < min(blocks, (run + 1) * each); ++b) a += __ldg(part + ((i64)b * sums + k) * d + c);
  s[run][lane] = a;
  __syncthreads();
  if (run || c >= d) return;
  for (int i = 1; i < 32; ++i) a += s[i][lane];
  if (outs.dtype[k] == OSSM_F32) put1(static_cast<float*>(outs.to[k]) + c, a);
  else if (outs.dtype[k] == OSSM_BF16) put1(static_cast<__nv_bfloat16*>(outs.to[k]) + c, a);
  else put1(static_cast<__half*>(outs.to[k]) + c, a);
}

// ---------------------------------------------------------------- host
inline size_t size_of(int t) { return t == OSSM_F32 ? 4 : 2; }

struct Plan {
  int R, N, per, at_once, blocks, sums;
  size_t bytes;
};
constexpr int kRingBytes = 208 << 10;
// Threads of a row: a warp up to 512 channels (8 rows a block), beyond that a
// block with 16 channels a thread; backward, which keeps up to five sums a
// channel in registers, 8 channels up to 2048 (with all five from 256 on).  (16384 x 2048, fp32 stream, two
// norms and a gate, side by side before two channels an instruction: 103 us forward
// with 8 channels a thread, 86 with 16; 197 and 219 us backward.)
inline Plan plan_of(const ossm_norm_args* a, bool bwd) {
  Plan q{};
  const int runs = (a->dim + 7) / 8;
  const bool full = a->post_norm || a->gate_kind;
  if (runs <= 32 || (runs <= 64 && !(bwd && full))) {
    q.N = runs <= 32 ? 1 : 2;
    q.R = 32;
    q.per = kWarpRows;
  } else {
    q.N = bwd && runs <= 256 ? 1 : 2;
    q.R = ((runs + q.N - 1) / q.N + 31) / 32 * 32;
    q.per = 1;
  }
  const i64 rows = std::max<i64>(1, (a->tokens + q.per - 1) / q.per);
  q.sums = full ? (int)kSums : a->grad_bias ? 2 : 1;
  // blocks that are at work at once: 512 threads an SM backward, 768 forward
  q.at_once = std::max(1, (bwd ? 512 : 768) / (q.R * q.per));
  q.blocks = (int)std::min<i64>(rows, (i64)q.at_once * device_sms());
  if (bwd) q.bytes = (size_t)q.blocks * q.sums * a->dim * 4;
  return q;
}

inline Params params_of(const ossm_norm_args* a, const Plan& q, bool bwd) {
  Params p{};
  const size_t sx = size_of(a->stream_dtype), sy = size_of(a->dtype);
  bool vec = a->dim % 8 == 0;
  auto rows = [&](const void* ptr, i64 st, size_t sz) {
    if (ptr && ((uintptr_t)ptr % 16 || st * sz % 16)) vec = false;
  };
  rows(a->x, a->x_stride, sx);
  rows(a->y, a->y_stride, sy);
  rows(a->r, bwd ? a->x_stride : a->dim, sx);
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
  p.gate_kind = a->gate_kind, p.gate = {a->gate, a->gate_dtype, nullptr}, p.gst = a->gate_stride;
  p.scale = a->scale, p.post = a->post_norm, p.norm = a->norm;
  p.w = {a->weight, a->weight_dtype, nullptr}, p.b = {a->bias, a->bias_dtype, nullptr};
  p.pw = {a->post_weight, a->post_weight_dtype, nullptr}, p.pb = {a->post_bias, a->post_bias_dtype, nullptr};
  auto aligned = [](const void* ptr) { return (uintptr_t)ptr % 16 == 0; };
  p.gate_vec = aligned(a->gate) && (a->gate_kind != OSSM_GATE_FULL || a->gate_stride * size_of(a->gate_dtype) % 16 == 0);
  p.w_vec = aligned(a->weight), p.b_vec = aligned(a->bias);
  p.pw_vec = aligned(a->post_weight), p.pb_vec = aligned(a->post_bias);
  p.post_eps = a->post_eps, p.eps = a->eps, p.inv_d = 1.f / a->dim;
  p.r = a->r, p.h = a->h, p.stats = a->stats;
  p.dr = a->grad_r, p.dh = a->grad_h, p.drst = a->grad_r_stride, p.dhst = a->grad_h_stride;
  p.status = a->status;
  p.dx = a->grad_x, p.dy = a->grad_y, p.dgate = a->grad_gate, p.dgate_dtype = a->gate_dtype;
  return p;
}

// The ring's stages, and the shared memory of a block: up to 8 rows ahead in
// what the blocks of an SM share.  Rows of which no two fit are read where they lie.
// row: bytes of a row of all tensors.
inline size_t ring_of(Params& p, const Plan& q, bool bwd, int row) {
  p.stage_bytes = row;
  const size_t stage = (size_t)row * q.per, most = kRingBytes / q.at_once;
  size_t shared = 4 * (size_t)p.d * ((p.w.p != nullptr) + (p.b.p != nullptr) + (p.pw.p != nullptr) +
                                     (p.pb.p != nullptr) + (p.gate_kind == G_CHANNEL));
  if (2 * stage > kRingBytes) p.vec = false;
  p.shared = shared + (p.vec ? 2 * stage : 0) <= most;
  if (!p.shared) shared = 0;
  p.stages = p.vec ? (int)std::max<size_t>(2, std::min<size_t>(kMaxStages, (most - std::min(most, shared)) / stage)) : 0;
  return std::max(p.stages * stage + shared, bwd && q.per > 1 ? (size_t)q.per * 8 * q.N * q.R * 4 : 0);
}

// Which of a kernel's six forms: 8 or 16 channels a thread, the most threads a
// block has.
inline int variant(const Params& p, const Plan& q) {
  if (p.vec) return q.N == 1 ? 0 : q.R <= 256 ? 1 : 2;
  return q.N == 1 ? 3 : q.R <= 256 ? 4 : 5;
}

template <typename TX, typename TY>
int forward(const ossm_norm_args* a, cudaStream_t st) {
  const Plan q = plan_of(a, false);
  Params p = params_of(a, q, false);
  const size_t smem = ring_of(p, q, false, p.d * (int)(sizeof(TX) + (a->y ? sizeof(TY) : 0)));
  const int which = variant(p, q);
  static constexpr void (*kerns[])(Params) = {
      norm_fwd_kernel<TX, TY, 1, true, 256>,  norm_fwd_kernel<TX, TY, 2, true, 256>,  norm_fwd_kernel<TX, TY, 2, true, 512>,
      norm_fwd_kernel<TX, TY, 1, false, 256>, norm_fwd_kernel<TX, TY, 2, false, 256>, norm_fwd_kernel<TX, TY, 2, false, 512>};
  static std::atomic<uint64_t> done[6];
  auto kern = kerns[which];
  if (allow_smem(kern, kRingBytes, done[which]) != cudaSuccess)
    return OSSM_ELAUNCH;
  kern<<<q.blocks, q.R * q.per, smem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

// N and MAXT by the plan.
template <typename TX, typename TY, int SUMS>
bool launch_bwd(const Plan& q, Params& p, cudaStream_t st) {
  const size_t smem = ring_of(p, q, true, p.d * (int)(sizeof(TX) + (p.dr ? sizeof(TX) : 0) + (p.dh ? sizeof(TY) : 0) +
                                                      (p.y ? sizeof(TY) : 0)));
  const int which = variant(p, q);
  static constexpr void (*kerns[])(Params) = {
      norm_bwd_kernel<TX, TY, 1, true, SUMS, 256>,  norm_bwd_kernel<TX, TY, 2, true, SUMS, 256>,
      norm_bwd_kernel<TX, TY, 2, true, SUMS, 512>,  norm_bwd_kernel<TX, TY, 1, false, SUMS, 256>,
      norm_bwd_kernel<TX, TY, 2, false, SUMS, 256>, norm_bwd_kernel<TX, TY, 2, false, SUMS, 512>};
  static std::atomic<uint64_t> done[6];
  auto kern = kerns[which];
  if (allow_smem(kern, kRingBytes, done[which]) != cudaSuccess)
    return false;
  kern<<<q.blocks, q.R * q.per, smem, st>>>(p);
  return true;
}

template <typename TX, typename TY>
int backward(const ossm_norm_args* a, const Plan& q, float* part, cudaStream_t st) {
  Params p = params_of(a, q, true);
  const bool sums = a->grad_weight || a->grad_bias || a->grad_post_weight || a->grad_post_bias ||
                    (a->gate_kind == OSSM_GATE_CHANNEL && a->grad_gate);
  p.part = sums ? part : nullptr;
  if (a->gate_kind == OSSM_GATE_CHANNEL) p.dgate = nullptr;
  if (!(q.sums == 1   ? launch_bwd<TX, TY, 1>(q, p, st)
        : q.sums == 2 ? launch_bwd<TX, TY, 2>(q, p, st)
                      : launch_bwd<TX, TY, kSums>(q, p, st)))
    return OSSM_ELAUNCH;
  if (sums) {
    Outs o{};
    o.to[S_W] = a->grad_weight, o.dtype[S_W] = a->weight_dtype;
    o.to[S_B] = a->grad_bias, o.dtype[S_B] = a->bias_dtype;
    if (a->gate_kind == OSSM_GATE_CHANNEL) o.to[S_GATE] = a->grad_gate, o.dtype[S_GATE] = a->gate_dtype;
    o.to[S_PW] = a->grad_post_weight, o.dtype[S_PW] = a->post_weight_dtype;
    o.to[S_PB] = a->grad_post_bias, o.dtype[S_PB] = a->post_bias_dtype;
    norm_sums_kernel<<<dim3((a->dim + 31) / 32, q.sums), 1024, 0, st>>>(part, q.blocks, q.sums, a->dim, o);
  }
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

}  // namespace nrm
}  // namespace ossm
