// Token embeddings, and their gradient by sorted tokens.
//
//   out_t = scale W[id_t], 0 where id_t is no row;  dW_v = scale sum_{id_t = v} g_t
//
// The gradient sorts the positions by token (a stable radix sort, so that the
// order of a sum is that of the positions), cuts the sorted list into chunks, a
// warp each, which add their rows up in fp32, and joins the sums of tokens that
// reach over several chunks in order: the result depends on nothing but the
// arguments.  Every row of dW is written once, untouched ones with zeros.
#include <cuda_fp16.h>

#include <algorithm>

#include "ossm_attn.cuh"

namespace ossm {
int device_sms();
namespace emb {

using attn::pack2;
using attn::to_f2;
typedef long long i64;

// ---------------------------------------------------------------- eight values at a time
template <typename T>
OSSM_DEV void load8(const T* p, float (&v)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const float2 a = to_f2<T>(u.x), b = to_f2<T>(u.y), c = to_f2<T>(u.z), d = to_f2<T>(u.w);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
template <>
OSSM_DEV void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
OSSM_DEV void store8(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <>
OSSM_DEV void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
OSSM_DEV float get1(const float* p) { return __ldg(p); }
OSSM_DEV float get1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
OSSM_DEV float get1(const __half* p) { return __half2float(*p); }
OSSM_DEV void put1(float* p, float v) { *p = v; }
OSSM_DEV void put1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
OSSM_DEV void put1(__half* p, float v) { *p = __float2half_rn(v); }

// ---------------------------------------------------------------- lookup
constexpr int kThreads = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    embed_fwd_kernel(const int64_t* ids, i64 tokens, int d, int V, const T* w, i64 wst, float scale, T* out) {
  const int per = VEC ? d / 8 : d;  // pieces of a row
  const i64 all = tokens * per, step = (i64)gridDim.x * kThreads;
  for (i64 i = (i64)blockIdx.x * kThreads + threadIdx.x; i < all; i += step) {
    const i64 t = i / per;
    const int e = (int)(i - t * per);
    const i64 id = __ldg(ids + t);
    const bool known = id >= 0 && id < V;
    if (VEC) {
      float v[8] = {};
      if (known) load8<T>(w + id * wst + 8 * e, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= scale;
      store8<T>(out + t * d + 8 * e, v);
    } else {
      put1(out + t * d + e, known ? get1(w + id * wst + e) * scale : 0.f);
    }
  }
}

// ---------------------------------------------------------------- sort by token
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = 8 * kThreads;  // of one step of a block
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kMaxSortBlocks = 128;

struct Sort {
  i64 T;
  int V, per;              // keys of a block, a multiple of kKeys
  int shift, bits;         // the digit
  const int64_t* ids;      // first pass: the tokens themselves
  const uint32_t *key, *pos;
  uint32_t *key_to, *pos_to;
  uint32_t* hist;          // [blocks][bins]
};
OSSM_DEV uint32_t key_of(const Sort& s, i64 i) {
  if (!s.ids) return s.key[i];
  const i64 id = __ldg(s.ids + i);
  return id >= 0 && id < s.V ? (uint32_t)id : (uint32_t)s.V;  // what is no row comes last
}

__global__ void __launch_bounds__(kThreads) embed_hist_kernel(const __grid_constant__ Sort s) {
  __shared__ uint32_t h[kMaxBins];
  const int bins = 1 << s.bits;
  for (int i = threadIdx.x; i < bins; i += kThreads) h[i] = 0;
  __syncthreads();
  const i64 a = (i64)blockIdx.x * s.per, b = min(s.T, a + s.per);
  for (i64 i = a + threadIdx.x; i < b; i += kThreads) atomicAdd(&h[(key_of(s, i) >> s.shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kThreads) s.hist[(i64)blockIdx.x * bins + i] = h[i];
}

__global__ void __launch_bounds__(kThreads) embed_scatter_kernel(const __grid_constant__ Sort s) {
  __shared__ uint32_t base[kMaxBins], sums[kWarps];
  __shared__ uint32_t count[kWarps][kMaxBins];
  const int bins = 1 << s.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // where this block's keys of each digit go: after all smaller digits, and the
  // same digit of earlier blocks
  uint32_t run = 0;
  for (int i0 = 0; i0 < bins; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    uint32_t before = 0, all = 0;
    if (i < bins)
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const uint32_t v = __ldg(s.hist + (i64)b * bins + i);
        all += v;
        before += b < (int)blockIdx.x ? v : 0;
      }
    uint32_t scan = all;
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const uint32_t u = __shfl_up_sync(~0u, scan, w);
      if (lane >= w) scan += u;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    uint32_t add = run;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) add += sums[w];
      run += sums[w];
    }
    if (i < bins) base[i] = add + scan - all + before;
  }
  const i64 a = (i64)blockIdx.x * s.per, b = min(s.T, a + s.per);
  for (i64 k0 = a; k0 < b; k0 += kKeys) {
    for (int i = threadIdx.x; i < kWarps * bins; i += kThreads) count[i / bins][i % bins] = 0;
    __syncthreads();
    uint32_t key[8], rank[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // a warp's keys lie side by side, in order
      const i64 i = k0 + warp * 256 + j * 32 + lane;
      const bool live = i < b;
      key[j] = live ? key_of(s, i) : 0;
      const uint32_t digit = live ? (key[j] >> s.shift) & (bins - 1) : kMaxBins + 1;
      const uint32_t same = __match_any_sync(~0u, digit);
      const uint32_t held = live ? count[warp][digit] : 0;
      rank[j] = held + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (live && lane == __ffs(same) - 1) count[warp][digit] = held + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += kThreads) {  // each warp's first place of a digit
      uint32_t at = base[i];
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t c = count[w][i];
        count[w][i] = at;
        at += c;
      }
      base[i] = at;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const i64 i = k0 + warp * 256 + j * 32 + lane;
      if (i < b) {
        const uint32_t to = count[warp][(key[j] >> s.shift) & (bins - 1)] + rank[j];
        s.key_to[to] = key[j];
        s.pos_to[to] = s.ids ? (uint32_t)i : s.pos[i];
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- sums
struct Sum {
  i64 T;
  int V, d, chunk, chunks, slices;
  const uint32_t *key, *pos;  // sorted
  i64 gst;
  float scale;
  float* part;  // [chunks][2][slices * kSlice]: of the token that began before the chunk, of the one that goes on after it
};
constexpr int kSlice = 512;     // channels of a warp: 16 a lane
constexpr int kZeroRows = 64;   // of a block that looks for untouched rows

OSSM_DEV i64 lower_bound(const uint32_t* key, i64 n, uint32_t v) {
  i64 lo = 0, hi = n;
  while (lo < hi) {
    const i64 mid = (lo + hi) >> 1;
    if (__ldg(key + mid) < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// A lane's 16 channels of a slice: two runs of eight, or every 32nd.
template <typename T, bool VEC>
struct Lane {
  int c0, d, lane;
  OSSM_DEV int at(int i) const { return VEC ? c0 + (i >> 3) * 256 + lane * 8 + (i & 7) : c0 + lane + 32 * i; }
  OSSM_DEV void add(const T* row, float (&v)[16]) const {
    if (VEC) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (at(8 * h) < d) {
          float u[8];
          load8<T>(row + at(8 * h), u);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[8 * h + i] += u[i];
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at(i) < d) v[i] += get1(row + at(i));
    }
  }
  OSSM_DEV void put(T* row, const float (&v)[16], float f) const {
    if (VEC) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (at(8 * h) < d) {
          float u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = v[8 * h + i] * f;
          store8<T>(row + at(8 * h), u);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (at(i) < d) put1(row + at(i), v[i] * f);
    }
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    embed_sum_kernel(const __grid_constant__ Sum s, const T* __restrict__ g, T* __restrict__ dw, int sum_blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= sum_blocks) {  // untouched rows
    __shared__ i64 range[2];
    __shared__ bool used[kZeroRows];
    const int v0 = (blockIdx.x - sum_blocks) * kZeroRows, v1 = min(s.V, v0 + kZeroRows);
    if (threadIdx.x < kZeroRows) used[threadIdx.x] = false;
    if (threadIdx.x < 64 && lane == 0) range[warp] = lower_bound(s.key, s.T, warp ? v1 : v0);
    __syncthreads();
    for (i64 i = range[0] + threadIdx.x; i < range[1]; i += kThreads) used[__ldg(s.key + i) - v0] = true;
    __syncthreads();
    const float zero[16] = {};
    for (int u = warp; u < (v1 - v0) * s.slices; u += kWarps) {
      const int v = u / s.slices;
      if (!used[v]) Lane<T, VEC>{u % s.slices * kSlice, s.d, lane}.put(dw + (i64)(v0 + v) * s.d, zero, 0.f);
    }
    return;
  }
  const i64 unit = (i64)blockIdx.x * kWarps + warp;
  const int slice = (int)(unit % s.slices);
  const i64 c = unit / s.slices;
  if (c >= s.chunks) return;
  const i64 a = c * s.chunk, b = min(s.T, a + s.chunk);
  const Lane<T, VEC> my{slice * kSlice, s.d, lane};
  float acc[16] = {};
  const uint32_t first = __ldg(s.key + a);
  uint32_t now = first;
  bool begun = a > 0 && __ldg(s.key + a - 1) == first;  // the token at hand began in an earlier chunk
  const uint32_t after = b < s.T ? __ldg(s.key + b) : ~0u;
  auto leave = [&](bool goes_on) {  // the token at hand is summed up
    if (now < (uint32_t)s.V) {
      if (begun || goes_on) {
        float* to = s.part + ((c * 2 + (begun ? 0 : 1)) * s.slices + slice) * kSlice;
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i * 32 + lane] = acc[i];
      } else {
        my.put(dw + (i64)now * s.d, acc, s.scale);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  };
  for (i64 i0 = a; i0 < b; i0 += 32) {
    const i64 i = min(i0 + lane, b - 1);
    const uint32_t keys = __ldg(s.key + i), poss = __ldg(s.pos + i);
    const int m = (int)min((i64)32, b - i0);
    for (int j = 0; j < m; ++j) {
      const uint32_t k = __shfl_sync(~0u, keys, j), t = __shfl_sync(~0u, poss, j);
      if (k != now) {
        leave(false);
        now = k;
        begun = false;
      }
      if (k < (uint32_t)s.V) my.add(g + (i64)t * s.gst, acc);
    }
  }
  leave(after == now);
}

// A block a chunk: the token that begins there and goes on, from its pieces in
// order, a run of them a warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    embed_join_kernel(const __grid_constant__ Sum s, T* __restrict__ dw) {
  __shared__ float sums[kWarps][kSlice];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const i64 c = blockIdx.x / s.slices;
  const int slice = blockIdx.x % s.slices;
  const i64 a = c * s.chunk, b = min(s.T, a + s.chunk);
  if (b >= s.T) return;
  const uint32_t k = __ldg(s.key + b - 1);
  if (k >= (uint32_t)s.V || __ldg(s.key + b) != k) return;             // does not go on
  if (a > 0 && __ldg(s.key + a) == k && __ldg(s.key + a - 1) == k) return;  // began before
  const i64 end = b + lower_bound(s.key + b, s.T - b, k + 1);           // past its last place
  const int pieces = (int)((end - 1) / s.chunk - c) + 1, each = (pieces + kWarps - 1) / kWarps;
  float acc[16] = {};
#pragma unroll 4
  for (int q = warp * each; q < min(pieces, (warp + 1) * each); ++q) {
    const float* from = s.part + (((c + q) * 2 + (q ? 0 : 1)) * s.slices + slice) * kSlice;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] += __ldg(from + i * 32 + lane);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) sums[warp][i * 32 + lane] = acc[i];
  __syncthreads();
  if (warp) return;
  for (int w = 1; w < kWarps; ++w)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] += sums[w][i * 32 + lane];
  Lane<T, VEC>{slice * kSlice, s.d, lane}.put(dw + (i64)k * s.d, acc, s.scale);
}

// ---------------------------------------------------------------- host
bool valid(const ossm_embed_args* a, bool bwd) {
  if (!a || a->tokens < 0 || a->tokens > (1LL << 31) - 1 || a->dim < 1 || a->dim > (1 << 16)) return false;
  if (a->vocab < 1 || a->vocab >= (1 << 27)) return false;
  if (a->dtype != OSSM_F32 && a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) return false;
  if (a->tokens && !a->ids) return false;
  if (bwd) return a->grad_weight && (a->tokens == 0 || (a->grad_out && a->grad_out_stride >= a->dim));
  return a->weight && a->weight_stride >= a->dim && (a->tokens == 0 || a->out);
}

struct Plan {
  int passes, bits, per, blocks, chunk, chunks, slices;
  size_t at[6], bytes;
};
Plan plan_of(const ossm_embed_args* a) {
  Plan q{};
  const i64 T = std::max<i64>(1, a->tokens);
  int bits = 1;
  while ((a->vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
  q.passes = (bits + kMaxBits - 1) / kMaxBits;
  q.bits = (bits + q.passes - 1) / q.passes;
  q.per = (int)((T + (i64)kKeys * kMaxSortBlocks - 1) / ((i64)kKeys * kMaxSortBlocks)) * kKeys;
  q.blocks = (int)((T + q.per - 1) / q.per);
  q.slices = (a->dim + kSlice - 1) / kSlice;
  // enough chunks for 32 warps an SM, of 8 to 64 positions
  q.chunk = (int)std::min<i64>(64, std::max<i64>(8, T * q.slices / (32 * (i64)device_sms())));
  q.chunks = (int)((T + q.chunk - 1) / q.chunk);
  size_t at = 0;
  int k = 0;
  auto take = [&](size_t bytes) {
    q.at[k++] = at;
    at += (bytes + 255) / 256 * 256;
  };
  for (int i = 0; i < 4; ++i) take(4 * T);  // keys and positions, twice
  take((size_t)q.blocks * 4 << q.bits);
  take((size_t)q.chunks * 2 * q.slices * kSlice * 4);
  q.bytes = at;
  return q;
}

template <typename T>
int forward(const ossm_embed_args* a, cudaStream_t st) {
  if (!a->tokens) return OSSM_OK;
  const T* w = static_cast<const T*>(a->weight);
  T* out = static_cast<T*>(a->out);
  constexpr int kUnit = 16 / sizeof(T);
  const bool vec = a->dim % 8 == 0 && a->weight_stride % kUnit == 0 && (uintptr_t)w % 16 == 0 && (uintptr_t)out % 16 == 0;
  const i64 all = a->tokens * (vec ? a->dim / 8 : a->dim);
  const int grid = (int)std::min<i64>((all + kThreads - 1) / kThreads, 16LL * device_sms());
  auto kern = vec ? embed_fwd_kernel<T, true> : embed_fwd_kernel<T, false>;
  kern<<<grid, kThreads, 0, st>>>(a->ids, a->tokens, a->dim, a->vocab, w, a->weight_stride, a->scale, out);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

template <typename T>
int backward(const ossm_embed_args* a, const Plan& q, char* w, cudaStream_t st) {
  if (!a->tokens)
    return cudaMemsetAsync(a->grad_weight, 0, (size_t)a->vocab * a->dim * sizeof(T), st) == cudaSuccess ? OSSM_OK
                                                                                                      : OSSM_ELAUNCH;
  uint32_t* buf[4];
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(w + q.at[i]);
  Sort s{};
  s.T = a->tokens, s.V = a->vocab, s.per = q.per, s.bits = q.bits;
  s.hist = reinterpret_cast<uint32_t*>(w + q.at[4]);
  for (int i = 0; i < q.passes; ++i) {
    s.shift = i * q.bits;
    s.ids = i ? nullptr : a->ids;
    s.key = buf[2 * (i & 1)], s.pos = buf[2 * (i & 1) + 1];
    s.key_to = buf[2 * (~i & 1)], s.pos_to = buf[2 * (~i & 1) + 1];
    embed_hist_kernel<<<q.blocks, kThreads, 0, st>>>(s);
    embed_scatter_kernel<<<q.blocks, kThreads, 0, st>>>(s);
  }
  const T* g = static_cast<const T*>(a->grad_out);
  T* dw = static_cast<T*>(a->grad_weight);
  Sum m{};
  m.T = a->tokens, m.V = a->vocab, m.d = a->dim, m.chunk = q.chunk, m.chunks = q.chunks, m.slices = q.slices;
  m.key = s.key_to, m.pos = s.pos_to, m.gst = a->grad_out_stride, m.scale = a->scale;
  m.part = reinterpret_cast<float*>(w + q.at[5]);
  constexpr int kUnit = 16 / sizeof(T);
  const bool vec = a->dim % 8 == 0 && a->grad_out_stride % kUnit == 0 && (uintptr_t)g % 16 == 0 && (uintptr_t)dw % 16 == 0;
  const int sum_blocks = (int)(((i64)q.chunks * q.slices + kWarps - 1) / kWarps);
  const int zero_blocks = (a->vocab + kZeroRows - 1) / kZeroRows;
  auto sum = vec ? embed_sum_kernel<T, true> : embed_sum_kernel<T, false>;
  auto join = vec ? embed_join_kernel<T, true> : embed_join_kernel<T, false>;
  sum<<<sum_blocks + zero_blocks, kThreads, 0, st>>>(m, g, dw, sum_blocks);
  if (q.chunks > 1) join<<<q.chunks * q.slices, kThreads, 0, st>>>(m, dw);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

}  // namespace emb
}  // namespace ossm

using namespace ossm;

extern "C" size_t ossm_embed_workspace_bytes(const ossm_embed_args* a) {
  return emb::valid(a, true) ? emb::plan_of(a).bytes : 0;
}
extern "C" int ossm_embed_fwd(const ossm_embed_args* a, ossm_stream_t stream) {
  if (!emb::valid(a, false)) return OSSM_EINVAL;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a->dtype == OSSM_F32    ? emb::forward<float>(a, st)
         : a->dtype == OSSM_BF16 ? emb::forward<__nv_bfloat16>(a, st)
                                 : emb::forward<__half>(a, st);
}
extern "C" int ossm_embed_bwd(const ossm_embed_args* a, void* workspace, size_t workspace_bytes, ossm_stream_t stream) {
  if (!emb::valid(a, true)) return OSSM_EINVAL;
  const emb::Plan q = emb::plan_of(a);
  if (!workspace || workspace_bytes < q.bytes || (uintptr_t)workspace % 256) return OSSM_EWORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(workspace);
  return a->dtype == OSSM_F32    ? emb::backward<float>(a, q, w, st)
         : a->dtype == OSSM_BF16 ? emb::backward<__nv_bfloat16>(a, q, w, st)
                                 : emb::backward<__half>(a, q, w, st);
}
extern "C" size_t ossm_sizeof_embed_args(void) { return sizeof(ossm_embed_args); }
