// Token embeddings, and their gradient by sorted tokens.
//
//   out_t = scale W[id_t], 0 where id_t is no row;  dW_v = scale sum_{id_t = v} g_t
//
// The gradient sorts the positions by token (a stable radix sort, so that the
// order of a sum is that of the positions), cuts the sorted list into chunks, a
// warp each, which add their rows up in fp32, and joins the sums of tokens that
// reach over several chunks in order: the result depends on nothing but the
// arguments.  dW is filled with zeros while the first digits are counted.
//
// What bounds it: lookup and sums move each byte once (131072 positions, 512
// channels, 32000 rows, bf16: 34 us, 7.9 TB/s with the rows in L2, and 32 us, 5.2
// TB/s); the sort, two digits, is 32 us of dependent launches, the joins 8.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

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
template <typename T>
OSSM_DEV void take8(const T* p, float (&v)[8]) {  // of registers
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = to_f2<T>(u.x), b = to_f2<T>(u.y), c = to_f2<T>(u.z), d = to_f2<T>(u.w);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
template <>
OSSM_DEV void take8<float>(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[i];
}
OSSM_DEV float get1(const float* p) { return *p; }
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
  if (!VEC) {  // rows that are not whole 16-byte pieces: a warp a token, 8 loads on their way
    const int lane = threadIdx.x & 31;
    for (i64 t = (i64)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < tokens; t += (i64)gridDim.x * (kThreads / 32)) {
      const i64 id = __ldg(ids + t);
      const bool known = id >= 0 && id < V;
      const T* const from = w + (known ? id * wst : 0);
      T* const to = out + t * d;
      for (int e0 = lane; e0 < d; e0 += 256) {
        T v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e0 + 32 * k < d) v[k] = from[e0 + 32 * k];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e0 + 32 * k < d) put1(to + e0 + 32 * k, known ? get1(&v[k]) * scale : 0.f);
      }
    }
    return;
  }
  const int per = d / 8;  // pieces of a row
  const i64 all = tokens * per, step = (i64)gridDim.x * kThreads;
  for (i64 i = (i64)blockIdx.x * kThreads + threadIdx.x; i < all; i += step) {
    const i64 t = i / per;
    const int e = (int)(i - t * per);
    const i64 id = __ldg(ids + t);
    float v[8] = {};
    if (id >= 0 && id < V) load8<T>(w + id * wst + 8 * e, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= scale;
    store8<T>(out + t * d + 8 * e, v);
  }
}

// ---------------------------------------------------------------- sort by token
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = 8 * kThreads;  // of one step of a block
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kMaxSortBlocks = 128;

struct Sort {
  i64 T;
  int V, per, blocks;      // keys of a block, a multiple of kKeys
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

// The blocks past s.blocks fill dW with zeros.
__global__ void __launch_bounds__(kThreads)
    embed_hist_kernel(const __grid_constant__ Sort s, char* __restrict__ dw, i64 dw_bytes) {
  __shared__ uint32_t h[kMaxBins];
  if ((int)blockIdx.x >= s.blocks) {
    char* const from = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(dw) + 15) & ~(uintptr_t)15);
    const i64 head = min((i64)(from - dw), dw_bytes), whole = (dw_bytes - head) / 16, tail = dw_bytes - head - 16 * whole;
    const i64 step = (i64)(gridDim.x - s.blocks) * kThreads, i0 = (i64)(blockIdx.x - s.blocks) * kThreads + threadIdx.x;
    for (i64 i = i0; i < whole; i += step) reinterpret_cast<uint4*>(from)[i] = make_uint4(0, 0, 0, 0);
    if (i0 < head) dw[i0] = 0;
    if (i0 < tail) from[16 * whole + i0] = 0;
    return;
  }
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
      for (int b0 = 0; b0 < s.blocks; b0 += 16) {  // 16 loads on their way
        uint32_t v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = b0 + k < s.blocks ? __ldg(s.hist + (i64)(b0 + k) * bins + i) : 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          all += v[k];
          before += b0 + k < (int)blockIdx.x ? v[k] : 0;
        }
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
  int V, d, chunk, chunks, slices, width;  // width: channels of a slice
  const uint32_t *key, *pos;  // sorted
  i64 gst;
  float scale;
  float* part;  // [chunks][2][slices * kSlice]: of the token that began before the chunk, of the one that goes on after it
};
constexpr int kSlice = 512;     // channels of a warp: 16 a lane
// A lane's 16 channels of a slice: two runs of eight, or every 32nd.
template <typename T, bool VEC>
struct Lane {
  int c0, d, lane;  // of channels c0 .. d
  OSSM_DEV int at(int i) const { return VEC ? c0 + (i >> 3) * 256 + lane * 8 + (i & 7) : c0 + lane + 32 * i; }
  OSSM_DEV bool has(int i) const { return at(VEC ? i & ~7 : i) < d; }
  struct alignas(16) Row {  // as it lies in memory
    T e[16];
  };
  OSSM_DEV void load(const T* row, Row& r) const {
    if (VEC) {
      constexpr int Q = sizeof(T) / 2;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (has(8 * h)) {
#pragma unroll
          for (int q = 0; q < Q; ++q)
            reinterpret_cast<uint4*>(r.e + 8 * h)[q] = __ldcs(reinterpret_cast<const uint4*>(row + at(8 * h)) + q);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (has(i)) r.e[i] = row[at(i)];
    }
  }
  OSSM_DEV void add(const Row& r, float (&v)[16]) const {  // past the row's end: anything, never stored
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float u[8];
      take8(r.e + 8 * h, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * h + i] += u[i];
    }
  }
  OSSM_DEV void put(T* row, const float (&v)[16], float f) const {
    if (VEC) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (has(8 * h)) {
          float u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = v[8 * h + i] * f;
          store8<T>(row + at(8 * h), u);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (has(i)) put1(row + at(i), v[i] * f);
    }
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    embed_sum_kernel(const __grid_constant__ Sum s, const T* __restrict__ g, T* __restrict__ dw) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const i64 unit = (i64)blockIdx.x * kWarps + warp;
  const int slice = (int)(unit % s.slices);
  const i64 c = unit / s.slices;
  if (c >= s.chunks) return;
  const i64 a = c * s.chunk, b = min(s.T, a + s.chunk);
  const Lane<T, VEC> my{slice * s.width, min(s.d, (slice + 1) * s.width), lane};
  float acc[16] = {};
  uint32_t keys = __ldg(s.key + min(a + lane, b - 1)), poss = __ldg(s.pos + min(a + lane, b - 1));
  const uint32_t before = a > 0 ? __ldg(s.key + a - 1) : ~0u, after = b < s.T ? __ldg(s.key + b) : ~0u;
  uint32_t now = __shfl_sync(~0u, keys, 0);
  bool begun = before == now;  // the token at hand began in an earlier chunk
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
  // kAhead rows on their way at a time; the positions of the next 32 too
  constexpr int kAhead = sizeof(T) == 4 || !VEC ? 4 : 8;
  for (i64 i0 = a; i0 < b; i0 += 32) {
    const int m = (int)min((i64)32, b - i0);
    const i64 next = min(i0 + 32 + lane, b - 1);
    const uint32_t keys_n = __ldg(s.key + next), poss_n = __ldg(s.pos + next);
    for (int j0 = 0; j0 < m; j0 += kAhead) {
      typename Lane<T, VEC>::Row row[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t k = __shfl_sync(~0u, keys, (j0 + j) & 31), t = __shfl_sync(~0u, poss, (j0 + j) & 31);
        if (j0 + j < m && k < (uint32_t)s.V) my.load(g + (i64)t * s.gst, row[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t k = __shfl_sync(~0u, keys, (j0 + j) & 31);
        if (j0 + j < m) {
          if (k != now) {
            leave(false);
            now = k;
            begun = false;
          }
          if (k < (uint32_t)s.V) my.add(row[j], acc);
        }
      }
    }
    keys = keys_n, poss = poss_n;
  }
  leave(after == now);
}

// Adds the pieces of tokens that go on over chunks up, in order.  A block looks
// through a run of chunks for those where such a token begins; a warp takes a
// token of up to 8 pieces, the block together one of more, a run of them a warp.
constexpr int kJoinThreads = 512, kJoinWarps = kJoinThreads / 32, kMaxRun = 512;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kJoinThreads)
    embed_join_kernel(const __grid_constant__ Sum s, T* __restrict__ dw, int run) {
  __shared__ float sums[kJoinWarps / 2][kSlice];
  __shared__ int begins[kMaxRun], longs[kMaxRun], nbegins, nlongs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.y;
  if (threadIdx.x == 0) nbegins = nlongs = 0;
  __syncthreads();
  const i64 c0 = (i64)blockIdx.x * run;
  for (int i = threadIdx.x; i < run && c0 + i < s.chunks; i += kJoinThreads) {
    const i64 a = (c0 + i) * s.chunk, b = a + s.chunk;
    if (b >= s.T) break;
    const uint32_t k = __ldg(s.key + b - 1), after = __ldg(s.key + b);
    const uint32_t before = a > 0 ? __ldg(s.key + a - 1) : ~0u;
    if (k < (uint32_t)s.V && after == k && before != k) begins[atomicAdd(&nbegins, 1)] = i;
  }
  __syncthreads();
  auto pieces_of = [&](i64 c, uint32_t k) {  // a warp: 1, and one for every later chunk that starts with the token
    int pieces = 1, n = 32;
    while (n == 32) {
      const i64 i = (c + pieces + lane) * s.chunk;
      n = __popc(__ballot_sync(~0u, i < s.T && __ldg(s.key + i) == k));
      pieces += n;
    }
    return pieces;
  };
  auto add = [&](i64 c, int from, int upto, float (&acc)[16]) {  // 4 pieces on their way
    for (int q0 = from; q0 < upto; q0 += 4) {
      float v[4][16];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int q = min(q0 + h, upto - 1);
        const float* p = s.part + (((c + q) * 2 + (q ? 0 : 1)) * s.slices + slice) * kSlice;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[h][i] = __ldg(p + i * 32 + lane);
      }
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (q0 + h < upto)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i] += v[h][i];
    }
  };
  auto token = [&](i64 c) { return __ldg(s.key + (c + 1) * s.chunk); };
  const Lane<T, VEC> my{slice * s.width, min(s.d, (slice + 1) * s.width), lane};
  for (int j = warp; j < nbegins; j += kJoinWarps) {
    const i64 c = c0 + begins[j];
    const uint32_t k = token(c);
    const int pieces = pieces_of(c, k);
    if (pieces > 8) {
      if (lane == 0) longs[atomicAdd(&nlongs, 1)] = begins[j];
      continue;
    }
    float acc[16] = {};
    add(c, 0, pieces, acc);
    my.put(dw + (i64)k * s.d, acc, s.scale);
  }
  __syncthreads();
  for (int j = 0; j < nlongs; ++j) {
    const i64 c = c0 + longs[j];
    const uint32_t k = token(c);
    const int pieces = pieces_of(c, k), each = (pieces + kJoinWarps - 1) / kJoinWarps;
    float acc[16] = {};
    add(c, min(pieces, warp * each), min(pieces, (warp + 1) * each), acc);
    for (int w = kJoinWarps / 2; w; w >>= 1) {  // halves of the warps
      __syncthreads();
      if (warp >= w && warp < 2 * w)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[warp - w][i * 32 + lane] = acc[i];
      __syncthreads();
      if (warp < w)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] += sums[warp][i * 32 + lane];
    }
    if (warp == 0) my.put(dw + (i64)k * s.d, acc, s.scale);
  }
}

// ---------------------------------------------------------------- host
bool valid(const ossm_embed_args* a, bool bwd) {
  if (!a || a->tokens < 0 || a->tokens > (1LL << 31) - 1 || a->dim < 1 || a->dim > (1 << 16)) return false;
  if (a->vocab < 1 || a->vocab >= (1 << 27)) return false;
  if (a->dtype != OSSM_F32 && a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) return false;
  if ((a->tokens && !a->ids) || !std::isfinite(a->scale)) return false;
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
  // a chunk for each of the 16 warps that an SM holds, of 8 positions at least
  const i64 warps = 16LL * device_sms();
  q.chunk = (int)std::max<i64>(8, (T * q.slices + warps - 1) / warps);
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
  const i64 all = vec ? a->tokens * (a->dim / 8) : 32 * a->tokens;
  const int grid = (int)std::min<i64>((all + kThreads - 1) / kThreads, 16LL * device_sms());
  auto kern = vec ? embed_fwd_kernel<T, true> : embed_fwd_kernel<T, false>;
  kern<<<grid, kThreads, 0, st>>>(a->ids, a->tokens, a->dim, a->vocab, w, a->weight_stride, a->scale, out);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

template <typename T>
int backward(const ossm_embed_args* a, const Plan& q, char* w, cudaStream_t st) {
  uint32_t* buf[4];
  for (int i = 0; i < 4; ++i) buf[i] = reinterpret_cast<uint32_t*>(w + q.at[i]);
  Sort s{};
  s.T = a->tokens, s.V = a->vocab, s.per = q.per, s.blocks = q.blocks, s.bits = q.bits;
  s.hist = reinterpret_cast<uint32_t*>(w + q.at[4]);
  for (int i = 0; i < (a->tokens ? q.passes : 1); ++i) {
    s.shift = i * q.bits;
    s.ids = i ? nullptr : a->ids;
    s.key = buf[2 * (i & 1)], s.pos = buf[2 * (i & 1) + 1];
    s.key_to = buf[2 * (~i & 1)], s.pos_to = buf[2 * (~i & 1) + 1];
    const i64 bytes = i ? 0 : (i64)a->vocab * a->dim * (i64)sizeof(T);
    const int zero = (int)std::min<i64>(4LL * device_sms(), (bytes + 16 * kThreads - 1) / (16 * kThreads));
    embed_hist_kernel<<<q.blocks + zero, kThreads, 0, st>>>(s, static_cast<char*>(a->grad_weight), bytes);
    if (a->tokens) embed_scatter_kernel<<<q.blocks, kThreads, 0, st>>>(s);
  }
  if (!a->tokens) return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
  const T* g = static_cast<const T*>(a->grad_out);
  T* dw = static_cast<T*>(a->grad_weight);
  Sum m{};
  m.width = ((a->dim + q.slices - 1) / q.slices + 7) / 8 * 8;
  m.T = a->tokens, m.V = a->vocab, m.d = a->dim, m.chunk = q.chunk, m.chunks = q.chunks, m.slices = q.slices;
  m.key = s.key_to, m.pos = s.pos_to, m.gst = a->grad_out_stride, m.scale = a->scale;
  m.part = reinterpret_cast<float*>(w + q.at[5]);
  constexpr int kUnit = 16 / sizeof(T);
  const bool vec = a->dim % 8 == 0 && a->grad_out_stride % kUnit == 0 && (uintptr_t)g % 16 == 0 && (uintptr_t)dw % 16 == 0;
  const int sum_blocks = (int)(((i64)q.chunks * q.slices + kWarps - 1) / kWarps);
  auto sum = vec ? embed_sum_kernel<T, true> : embed_sum_kernel<T, false>;
  auto join = vec ? embed_join_kernel<T, true> : embed_join_kernel<T, false>;
  sum<<<sum_blocks, kThreads, 0, st>>>(m, g, dw);
  if (q.chunks > 1) {
    const int run = (int)std::min<i64>(kMaxRun, std::max<i64>(8, (q.chunks + 2LL * device_sms() - 1) / (2LL * device_sms())));
    join<<<dim3((q.chunks + run - 1) / run, q.slices), kJoinThreads, 0, st>>>(m, dw, run);
  }
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
