// The next token of each row from given random numbers (ossm_sample_tokens).
//
// Every filter keeps a prefix of the candidates ordered by (logit descending,
// index ascending), so what stays is described by one 64-bit key: the logit's
// order-preserving bits above the inverted index.
//
// A row is shared by a cluster of up to 8 CTAs.  One pass over the logits finds
// the largest and the sum of the weights, from which follows a logit that the
// prefix cannot reach below (Bound); a second pass, out of L2, collects the
// candidates above it into the first CTA's shared memory, where the prefix's end
// and its best score are found: a few candidates in order, of more a histogram
// first.  The noise is read for the prefix alone.  In wide rows the bound is
// guessed from a sample and the guess checked by the mass collected.  Where too
// many candidates are collected all the same (nearly flat rows) the first CTA
// goes over the row instead of the list.
// Masses that are compared, the whole row's among them, are 64-bit fixed-point
// sums of one function of the logit: they do not depend on the order of the
// additions, nor on how many CTAs a row gets.  (The fp32 sum of the first pass
// gives the bound and the guess alone.)
// Measured back to back, replayed from a graph (a call among others takes 1 to 2
// us more): 1 x 32000 bf16, top-k 50 and top-p 0.95: 11.2 us; 128 x 131072 bf16,
// top-k 50: 16.5 us (5.1 us of reads), min-p 0.01: 18.7 us, top-p 0.72 (4000
// stay): 42 us, top-p 0.92 (18000 stay): 63 us.  What bounds it there: one CTA an
// SM works through steps that wait for one another; of 49 us of a row whose list
// is 12000 long, 7.5 are the first pass (5 of reads), 5 the sample, 16 the
// collection with the row's mass (6 of them the mass), 11 the prefix's end, 6 the
// noise.  64 registers a thread, with 32 (fp32) to 52 bytes spilled.
//
// Without filters the score of every candidate is needed: one pass over logits
// and noise.  The logarithm is first taken in its fast form, and exactly only
// where that comes within its error of the best score so far.
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "orthossm_b200.h"
#include "ossm_common.cuh"

namespace ossm {
int device_sms();
namespace smp {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kOpen = 512;     // threads of a CTA where nothing is filtered
constexpr int kList = 24576;   // candidates that shared memory holds
constexpr int kRank = 256;     // candidates that are put in order
constexpr int kBins = 1024;
constexpr int kGuess = 4096;   // logits a CTA from which on a guess of the bound pays
typedef unsigned long long u64;
typedef long long i64;

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
constexpr float kLowest = -3.402823466e38f;  // the lowest candidate

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

OSSM_DEV int index_of(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

// Probability relative to the first candidate (logit m): 1 at l == m, also
// where both are +inf.
OSSM_DEV float weight(float l, float m, float inv_t) {
  return l == m ? 1.f : expf(__fmul_rn(__fsub_rn(l, m), inv_t));
}
OSSM_DEV float ex2(float x) {  // 2^x, relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
OSSM_DEV float2 add2(float2 a, float2 b) { return fma2(a, make_float2(1.f, 1.f), b); }
// Masses: the candidates' weights (0 to 1, relative to the row's largest logit m)
// in steps of 2^-40, to the nearest; a row's sum stays below 2^63 for V < 2^23
// equal candidates.  Everything that is compared is a sum of these, the whole
// row's mass too, so that the prefix's end does not depend on how a row is
// divided, nor on which of the ways below finds it.
constexpr float kRound = 64.f, kRound2 = 0x1.8p-17f;  // numbers next to these are 2^-17 and 2^-40 apart
struct Masses {
  float m, c, c_lo, least;  // c + c_lo = log2(e) / temperature; logits further below m weigh nothing
  OSSM_DEV Masses(float m, float inv_t) : m(m) {
    constexpr float kL = 1.44269504f, kL_lo = 1.92596303e-8f;  // log2(e)
    const float x = inv_t * kL;
    c = fminf(x, 3e38f);
    c_lo = x == c ? fmaf(inv_t, kL_lo, fmaf(inv_t, kL, -x)) : 0.f;
    least = fmaxf(-64.f / c, kLowest);
  }
  // The steps of 2^-17 are rounded off by one addition, then what is left in
  // steps of 2^-40 by a second: exact.
  OSSM_DEV u64 of(float l) const {
    const float d = l == m ? 0.f : fmaxf(__fsub_rn(l, m), least);
    const float w = ex2(__fmaf_rn(d, c, __fmul_rn(d, c_lo)));
    const float h = __fadd_rn(w, kRound), y = __fadd_rn(__fsub_rn(w, __fsub_rn(h, kRound)), kRound2);
    const int hi = __float_as_int(h) - __float_as_int(kRound), lo = __float_as_int(y) - __float_as_int(kRound2);
    return ((u64)hi << 23) + (i64)lo;
  }
  // The sum over N logits (m finite; what is no candidate weighs nothing),
  // added to h and y: the two roundings' bits, kRound's and kRound2's included.
  template <int N>
  OSSM_DEV void add(const float (&l)[N], uint32_t& h, uint32_t& y) const {
    const float2 m2 = make_float2(m, m), c2 = make_float2(c, c), lo2 = make_float2(c_lo, c_lo);
    const float2 r1 = make_float2(kRound, kRound), r2 = make_float2(kRound2, kRound2);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float2 d = sub2(make_float2(l[e], l[e + 1]), m2);
      d = make_float2(fmaxf(d.x, least), fmaxf(d.y, least));  // a NaN operand loses
      d = fma2(d, c2, mul2(d, lo2));
      const float2 w = make_float2(ex2(d.x), ex2(d.y));
      const float2 a = add2(w, r1), b = add2(sub2(w, sub2(a, r1)), r2);
      h += __float_as_uint(a.x) + __float_as_uint(a.y);
      y += __float_as_uint(b.x) + __float_as_uint(b.y);
    }
  }
  static OSSM_DEV u64 sum(uint32_t h, uint32_t y, int n) {  // of n logits added, n <= 2^8
    h -= n * __float_as_uint(kRound);
    y -= n * __float_as_uint(kRound2);
    return ((u64)h << 23) + (i64)(int)y;
  }
};

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

template <typename T>
struct Vec {
  static constexpr int n = 16 / sizeof(T);
};
OSSM_DEV void unpack(const uint4& u, float (&l)[4], float) {
  l[0] = __uint_as_float(u.x), l[1] = __uint_as_float(u.y), l[2] = __uint_as_float(u.z), l[3] = __uint_as_float(u.w);
}
OSSM_DEV void unpack(const uint4& u, float (&l)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    l[2 * i] = __uint_as_float(w[i] << 16), l[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
OSSM_DEV void unpack(const uint4& u, float (&l)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    l[2 * i] = f.x, l[2 * i + 1] = f.y;
  }
}

// Number e of a vector.
OSSM_DEV float pick(const uint4& u, int e, float) {
  return __uint_as_float(e & 2 ? (e & 1 ? u.w : u.z) : (e & 1 ? u.y : u.x));
}
OSSM_DEV uint32_t half_of(const uint4& u, int e) {
  const uint32_t w = e & 4 ? (e & 2 ? u.w : u.z) : (e & 2 ? u.y : u.x);
  return e & 1 ? w >> 16 : w & 0xffffu;
}
OSSM_DEV float pick(const uint4& u, int e, __nv_bfloat16) { return __uint_as_float(half_of(u, e) << 16); }
OSSM_DEV float pick(const uint4& u, int e, __half) {
  return __half2float(__ushort_as_half((unsigned short)half_of(u, e)));
}

// This CTA's share of a row: vectors v0 to v1 of 16 aligned bytes from logit
// `head` on.
template <typename T>
struct Share {
  const uint4* body;
  int head, nv, v0, v1;
  OSSM_DEV Share(const T* row, int V, int rank, int nrank) {
    head = min(V, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
    nv = (V - head) / Vec<T>::n;
    v0 = (int)((i64)nv * rank / nrank), v1 = (int)((i64)nv * (rank + 1) / nrank);
    body = reinterpret_cast<const uint4*>(row + head);
  }
};

// This CTA's share of a row: f(l, i, n) for the n logits from index i on, 16
// aligned bytes at a time; the row's unaligned ends go to the first CTA, one by
// one.  What is not a candidate (NaN) arrives as -inf.
template <typename T, typename F>
OSSM_DEV void scan(const T* row, int V, int rank, int nrank, F f) {
  constexpr int N = Vec<T>::n;
  const Share<T> own(row, V, rank, nrank);
  const int head = own.head, nv = own.nv, v0 = own.v0, v1 = own.v1;
  const uint4* body = own.body;
  for (int v = v0 + threadIdx.x; v < v1; v += 4 * kThreads) {
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (v + k * kThreads < v1) u[k] = __ldg(body + v + k * kThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (v + k * kThreads >= v1) break;
      float l[N];
      unpack(u[k], l, T());
#pragma unroll
      for (int e = 0; e < N; ++e) l[e] = fmaxf(l[e], -INFINITY);  // a NaN operand loses
      f(l, head + (v + k * kThreads) * N, N);
    }
  }
  if (rank == 0) {
    const int tail = V - head - nv * N, e = threadIdx.x;
    if (e < head + tail) {
      const int i = e < head ? e : V - tail + (e - head);
      float l[N];
      l[0] = fmaxf(to_f(row[i]), -INFINITY);
      f(l, i, 1);
    }
  }
}

// The same with the noise of each logit: f(l, e, i, n), by all lanes of a warp
// together (n = 0: nothing for this lane).  Both are loaded ahead for several
// vectors, as the noise comes from HBM.
template <int NT, typename T, typename F>
OSSM_DEV void scan_noise(const T* row, const float* nz, int V, int rank, int nrank, F f) {
  constexpr int N = Vec<T>::n, U = 16 / N;
  const Share<T> own(row, V, rank, nrank);
  const int head = own.head, nv = own.nv, v0 = own.v0, v1 = own.v1;
  const uint4* body = own.body;
  const float* nbody = nz + head;
  const bool aligned = ((uintptr_t)nbody & 15) == 0;
  const int lane = threadIdx.x & 31;
  for (int v = v0 + (threadIdx.x - lane); v < v1; v += U * NT) {  // of the warp's first lane
    uint4 u[U];
    float e[U][N];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int w = v + lane + k * NT;
      if (w >= v1) break;
      u[k] = __ldg(body + w);
      if (aligned) {
#pragma unroll
        for (int h = 0; h < N; h += 4) {
          const float4 x = __ldcs(reinterpret_cast<const float4*>(nbody + (size_t)w * N + h));
          e[k][h] = x.x, e[k][h + 1] = x.y, e[k][h + 2] = x.z, e[k][h + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int h = 0; h < N; ++h) e[k][h] = __ldcs(nbody + (size_t)w * N + h);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (v + k * NT >= v1) break;
      const int w = v + lane + k * NT;
      float l[N];
      unpack(u[k], l, T());
#pragma unroll
      for (int h = 0; h < N; ++h) l[h] = fmaxf(l[h], -INFINITY);
      f(l, e[k], head + w * N, w < v1 ? N : 0);
    }
  }
  if (rank == 0 && threadIdx.x < 32) {  // the ends: fewer than 16 logits
    const int tail = V - head - nv * N, n = lane < head + tail ? 1 : 0;
    const int i = lane < head ? lane : V - tail + (lane - head);
    float l[N], e[N];
    if (n) l[0] = fmaxf(to_f(row[i]), -INFINITY), e[0] = nz[i];
    f(l, e, i, n);
  }
}

template <typename V, typename Op>
OSSM_DEV V block_reduce(V v, V* red, Op op) {  // the result in every thread
#pragma unroll
  for (int w = 16; w; w >>= 1) v = op(v, __shfl_xor_sync(~0u, v, w));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
#pragma unroll
  for (int w = 16; w; w >>= 1) v = op(v, __shfl_xor_sync(~0u, v, w));
  return v;
}

template <int NT>
OSSM_DEV Best block_best(Best b, Best* bests) {  // the result in warp 0
  for (int w = 16; w; w >>= 1) better(b, __shfl_xor_sync(~0u, b.s, w), __shfl_xor_sync(~0u, b.i, w));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) bests[threadIdx.x >> 5] = b;
  __syncthreads();
  b = bests[threadIdx.x & (NT / 32 - 1)];
  for (int w = 16; w; w >>= 1) better(b, __shfl_xor_sync(~0u, b.s, w), __shfl_xor_sync(~0u, b.i, w));
  return b;
}

// A row's settings, in force together.
struct Row {
  float inv_t, top_p, min_p;
  int top_k;     // 0: off
  bool greedy;   // the first candidate alone
  OSSM_DEV bool open() const { return !greedy && top_k == 0 && top_p >= 1.f && !(min_p > 0.f); }
};
OSSM_DEV Row row_of(const Params& p, int row) {
  Row r;
  r.inv_t = p.inv_t;
  if (p.t_row) {  // not below the least fp32 number: 0 is the largest logit alone
    const float t = p.t_row[row];
    r.inv_t = t > 0.f ? fmaxf(1.0f / t, 0x1p-149f) : 0.f;
  }
  r.top_k = p.k_row ? p.k_row[row] : p.top_k;
  r.top_p = p.p_row ? p.p_row[row] : p.top_p;
  r.min_p = p.m_row ? p.m_row[row] : p.min_p;
  if (r.top_k <= 0 || r.top_k >= p.V) r.top_k = 0;
  if (!(r.top_p >= 0.f)) r.top_p = 0.f;
  r.greedy = !p.noise || !(r.inv_t > 0.f) || r.inv_t == INFINITY || r.min_p > 1.f;
  return r;
}

// Shared memory of the work on one row.
struct Room {
  u64 list[kList];
  u64 bins[kBins];
  u64 few[kRank];
  u64 red[32];
  u64 sh[4];
};

// The n <= kRank keys of a list in descending order: a key's position is the
// number of larger ones; parts of the count by neighbouring threads.
OSSM_DEV void order(u64* list, int n) {
  const int tid = threadIdx.x;
  int parts = 1;
  while (parts < 32 && n * parts * 2 <= kThreads) parts *= 2;
  const int e = tid / parts, q = tid % parts;
  u64 key = 0;
  int larger = 0;
  if (e < n) {
    key = list[e];
#pragma unroll 8
    for (int k = q; k < n; k += parts) larger += list[k] > key;
  }
  for (int w = 1; w < parts; w *= 2) larger += __shfl_xor_sync(~0u, larger, w);
  __syncthreads();
  if (e < n && q == 0) list[larger] = key;
  __syncthreads();
}

// Sum of v over the threads up to and including this one; all: over every thread.
OSSM_DEV u64 block_scan(u64 v, u64* red, u64& all) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int w = 1; w < 32; w *= 2) {
    const u64 u = __shfl_up_sync(~0u, v, w);
    if ((tid & 31) >= w) v += u;
  }
  __syncthreads();
  if ((tid & 31) == 31) red[tid >> 5] = v;
  __syncthreads();
  u64 before = (tid & 31) < (tid >> 5) ? red[tid & 31] : 0;
  all = red[tid & 31];
#pragma unroll
  for (int w = 16; w; w >>= 1) {
    before += __shfl_xor_sync(~0u, before, w);
    all += __shfl_xor_sync(~0u, all, w);
  }
  return before + v;
}

OSSM_DEV u64 share(float top_p, u64 whole) {  // the mass that a prefix has to reach
  return max((u64)1, (u64)__double2ull_ru((double)top_p * (double)whole));
}
// How many of n <= kRank keys in order the prefix holds (at least one) whose
// mass reaches `target`, or (target == 0) the share top_p of theirs; n + 1: they
// do not reach it.
OSSM_DEV int reaching(const u64* list, int n, const Masses& ms, const Row& r, u64 target, u64* red) {
  const int tid = threadIdx.x;
  const u64 own = tid < n ? ms.of(logit_of(list[tid])) : 0;
  u64 all;
  const u64 upto = block_scan(own, red, all);
  if (target == 0) target = share(r.top_p, all);
  const int stay = max(1, __syncthreads_count(tid < n && upto - own < target));
  return all < target ? n + 1 : stay;
}

// A 64-bit sum in shared memory of 32-bit atomics: one with a result, a second
// where it carries or q has a high part.  (A 64-bit one is a loop of exchanges.)
OSSM_DEV void add64(u64* to, u64 q) {
  uint32_t* w = reinterpret_cast<uint32_t*>(to);
  const uint32_t lo = (uint32_t)q, old = atomicAdd(w, lo), hi = (uint32_t)(q >> 32) + (old + lo < old);
  if (hi) atomicAdd(w + 1, hi);
}

OSSM_DEV void clear_bins(Room& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins[i] = 0;
  __syncthreads();
}
// The bin in which the sums of s.bins, from the first on, reach `target`, or
// (target == 0) the share top_p of them all; -1: none.  left: what of it the bin
// itself has to give.
OSSM_DEV int find_bin(Room& s, u64 target, float top_p, u64& left) {
  static_assert(kBins == kThreads, "a bin a thread");
  __syncthreads();
  const u64 own = s.bins[threadIdx.x];
  u64 all;
  const u64 upto = block_scan(own, s.red, all);
  if (target == 0) target = share(top_p, all);
  if (threadIdx.x == 0) s.sh[0] = ~(u64)0;
  __syncthreads();
  if (upto - own < target && target <= upto) {
    s.sh[0] = threadIdx.x;
    s.sh[1] = target - (upto - own);
  }
  __syncthreads();
  const int bin = (int)s.sh[0];
  left = s.sh[1];
  __syncthreads();
  return bin;
}

// The smallest key of the prefix of a set of keys that holds `left` of them
// (count) or of their mass; each(f) calls f for every key of the set.  As long
// as more than kRank are between the bounds, their range is cut into bins and
// narrowed to the one where the prefix ends; keys differ, so that ends.
template <typename Each>
OSSM_DEV u64 narrow(const Row& r, Each each, bool count, u64 left, const Masses& ms, Room& s) {
  u64 lo = 0, hi = ~(u64)0;
  int* fill = reinterpret_cast<int*>(&s.sh[3]);
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) *fill = 0;
    __syncthreads();
    u64 least = ~(u64)0, most = 0;
    int at = 0;
    each([&](u64 key) {
      if (key < lo || key > hi) return;
      if (at < kRank && (at = atomicAdd(fill, 1)) < kRank) s.few[at] = key;
      least = min(least, key), most = max(most, key);
    });
    __syncthreads();
    const int n = *fill;
    if (n <= kRank) {
      order(s.few, n);
      return s.few[(count ? (int)left : min(n, reaching(s.few, n, ms, r, left, s.red))) - 1];
    }
    lo = block_reduce(least, s.red, [](u64 a, u64 b) { return min(a, b); });
    hi = block_reduce(most, s.red, [](u64 a, u64 b) { return max(a, b); });
    const int shift = max(0, 54 - __clzll((long long)(hi - lo)));
    clear_bins(s);
    each([&](u64 key) {
      if (key >= lo && key <= hi)
        add64(s.bins + ((hi - key) >> shift), count ? 1 : ms.of(logit_of(key)));
    });
    const int bin = find_bin(s, left, 1.f, left);
    if (bin < 0) return lo;
    hi -= (u64)bin << shift;
    const u64 width = ((u64)1 << shift) - 1;
    lo = max(lo, hi > width ? hi - width : 0);
  }
}

// A logit's bin between the largest, m, and lb: (m - l) scale, rounded by adding
// 2^23, in the low bits.
struct Bins {
  float m, scale;
  OSSM_DEV Bins(float m, float lb) : m(m), scale(m > lb && m - lb < INFINITY ? (kBins - 1) / (m - lb) : 0.f) {}
  OSSM_DEV float below(float l) const { return l == m ? 0.f : m - l; }
  OSSM_DEV int of(float d) const {
    return __float_as_int(fminf(d * scale, (float)(kBins - 1)) + 8388608.f) & (kBins - 1);
  }
};

// The smallest key of the prefix of the list's N candidates at or above `floor`
// that holds `count` of them, or (count == 0) the mass `target` (0: the share
// top_p of theirs); `floor` where they do not reach it.
OSSM_DEV u64 select_list(const Row& r, int N, const Masses& ms, u64 floor, int count, u64 target, Room& s) {
  auto all = [&](auto f) {
    for (int e = threadIdx.x; e < N; e += kThreads)
      if (s.list[e] >= floor) f(s.list[e]);
  };
  u64 least = ~(u64)0;
  all([&](u64 key) { least = min(least, key); });
  const Bins bins(ms.m, logit_of(block_reduce(least, s.red, [](u64 a, u64 b) { return min(a, b); })));
  clear_bins(s);
  all([&](u64 key) {
    const float l = logit_of(key);
    add64(s.bins + bins.of(bins.below(l)), count ? 1 : ms.of(l));
  });
  u64 left;
  const int cut = find_bin(s, count ? (u64)count : target, r.top_p, left);
  if (cut < 0) return floor;  // all of them stay
  auto each = [&](auto f) {
    all([&](u64 key) {
      if (bins.of(bins.below(logit_of(key))) == cut) f(key);
    });
  };
  return narrow(r, each, count != 0, left, ms, s);
}

// The same of all the row's candidates, by one CTA; `whole`: their mass where it
// is known, else 0.  Candidates below logit lb are known to lie behind the
// prefix.
template <typename T>
OSSM_DEV u64 select_row(const Row& r, const T* lg, int V, const Masses& ms, float lb, u64 floor, int count, u64 whole,
                        Room& s) {
  const float m = ms.m;
  const Bins bins(m, lb);
  const float first = floor ? logit_of(floor) : -INFINITY;  // floor's logit: only there the index decides
  const float low = fmaxf(lb, kLowest);
  uint32_t* part = reinterpret_cast<uint32_t*>(s.bins);  // counts: the low half of a bin's sum
  clear_bins(s);
  scan(lg, V, 0, 1, [&](const float* l, int i, int n) {
#pragma unroll
    for (int e = 0; e < Vec<T>::n; ++e) {
      const bool in = e < n && l[e] >= low && (l[e] > first || key_of(l[e], i + e) >= floor);
      const int b = bins.of(bins.below(l[e]));
      if (!in) continue;
      if (count)
        atomicAdd(part + 2 * b, 1u);
      else
        add64(s.bins + b, ms.of(l[e]));
    }
  });
  u64 left;
  const int cut = find_bin(s, count ? (u64)count : whole ? share(r.top_p, whole) : 0, r.top_p, left);
  if (cut < 0) return floor;  // all of them stay
  // the bin's logits lie between these (half a bin wider on both sides)
  const float scale = bins.scale;
  const float from = scale > 0.f ? fmaxf(low, cut == kBins - 1 ? low : m - (cut + 1.f) / scale) : low;
  const float to = scale > 0.f && cut ? m - (cut - 1.f) / scale : INFINITY;
  auto each = [&](auto f) {  // the keys of the bin
    scan(lg, V, 0, 1, [&](const float* l, int i, int n) {
#pragma unroll
      for (int e = 0; e < Vec<T>::n; ++e)
        if (e < n && l[e] >= from && l[e] <= to && bins.of(bins.below(l[e])) == cut) {
          const u64 key = key_of(l[e], i + e);
          if (key >= floor) f(key);
        }
    });
  };
  int* fill = reinterpret_cast<int*>(&s.sh[2]);
  if (threadIdx.x == 0) *fill = 0;
  __syncthreads();
  int at = 0;
  each([&](u64 key) {
    if (at < kList && (at = atomicAdd(fill, 1)) < kList) s.list[at] = key;
  });
  __syncthreads();
  const int size = *fill;
  if (size > kList) return narrow(r, each, count != 0, left, ms, s);
  auto listed = [&](auto f) {
    for (int e = threadIdx.x; e < size; e += kThreads) f(s.list[e]);
  };
  return narrow(r, listed, count != 0, left, ms, s);
}

// The candidates of this CTA's share from logit `low` on, into a list; *count may
// pass the list's end, which is then found in another way.  A warp's four
// vectors take their places with one addition, and the candidates are walked
// by the bits set: code for each of the 32 logits of a thread ran in every warp
// that had one candidate (128 rows of 131072, 4000 candidates each, before the masses were added up here: 43 us, so 37).
// With `sum` it also returns the mass that this thread has seen of the share.
template <bool sum, typename T>
OSSM_DEV u64 collect(const T* row, int V, int rank, int nrank, float low, const Masses& ms, int* count, u64* list) {
  constexpr int N = Vec<T>::n, U = 4;
  const Share<T> own(row, V, rank, nrank);
  const int lane = threadIdx.x & 31;
  bool over = false;
  u64 mass = 0;
  for (int first = own.v0; first < own.v1 && !(over && !sum); first += U * kThreads) {
    const int v = first + threadIdx.x;
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (v + k * kThreads < own.v1) u[k] = __ldg(own.body + v + k * kThreads);
    uint32_t in = 0, h = 0, y = 0;
    int n = 0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (v + k * kThreads >= own.v1) break;
      float l[N];
      unpack(u[k], l, T());
#pragma unroll
      for (int e = 0; e < N; ++e) in |= l[e] >= low ? 1u << (k * N + e) : 0u;  // a NaN is not
      if (sum) ms.add(l, h, y);
      n += N;
    }
    if (sum) mass += Masses::sum(h, y, n);
    if (over || !__any_sync(~0u, in)) continue;
    int upto = __popc(in);
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const int x = __shfl_up_sync(~0u, upto, w);
      if (lane >= w) upto += x;
    }
    int at = lane == 31 ? atomicAdd(count, upto) : 0;
    at = __shfl_sync(~0u, at, 31);
    over = at >= kList;
    at += upto - __popc(in);
#pragma unroll
    for (int k = 0; k < U; ++k)
      for (uint32_t left = in >> (k * N) & ((1u << N) - 1); left; left &= left - 1, ++at) {
        const int e = __ffs(left) - 1;
        if (at < kList) list[at] = key_of(pick(u[k], e, T()), own.head + (v + k * kThreads) * N + e);
      }
  }
  if (rank == 0) {
    const int tail = V - own.head - own.nv * N, e = threadIdx.x;
    if (e < own.head + tail) {
      const int i = e < own.head ? e : V - tail + (e - own.head);
      const float l = to_f(row[i]);
      if (l >= low) {
        const int at = atomicAdd(count, 1);
        if (at < kList) list[at] = key_of(l, i);
      }
      if (sum && live(l)) mass += ms.of(l);
    }
  }
  return mass;
}

// A guess of the logit below which this CTA's share of the row holds `tail` of
// mass: from up to 16 logits a thread, spread over the share, a histogram
// between lb (known to lie below) and m.  In whole steps, so that the guess does
// not depend on the order of the additions either.
template <typename T>
OSSM_DEV float guess_bound(const T* lg, int V, int rank, int nrank, float m, float lb, float c, float tail, Room& s) {
  constexpr int N = Vec<T>::n, U = 16 / N;
  const Bins bins(m, lb);
  const Share<T> own(lg, V, rank, nrank);
  const int nv = own.v1 - own.v0, read = min(nv, U * kThreads);
  uint32_t* part = reinterpret_cast<uint32_t*>(s.bins);
  clear_bins(s);
  const float scale = 0x1p22f * ((float)nv / read) / tail;  // the sums: 2^22 where the sample's tail is reached
  uint32_t last = 0;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int at = threadIdx.x + k * kThreads;
    if (at >= read) continue;
    float l[N];
    unpack(__ldg(own.body + own.v0 + (int)((i64)at * nv / read)), l, T());
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = bins.below(fmaxf(l[e], -INFINITY));
      // at most 2^17 each, of 2^14 logits: a sum of 32 bits holds them
      const uint32_t q = __float2uint_rn(fminf(ex2(-d * c) * scale, 0x1p17f));
      const int b = bins.of(d);
      if (b == kBins - 1)
        last += q;  // most of them, perhaps
      else
        atomicAdd(part + 2 * b, q);
    }
  }
  last = __reduce_add_sync(~0u, last);
  if ((threadIdx.x & 31) == 0) atomicAdd(part + 2 * (kBins - 1), last);
  __syncthreads();
  u64 all;
  const u64 upto = block_scan(part[2 * threadIdx.x], s.red, all);
  const int bin = __syncthreads_count(all - upto > (u64)(0.9f * 0x1p22f));
  return bin >= kBins - 1 ? lb : fmaxf(lb, m - (bin + 0.5f) / bins.scale);
}

OSSM_DEV float lg2(float x) {  // log2, within 2^-22 (of 1, or of its value)
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The scores of a vector's logits l >= low that are candidates (stays(l, i))
// against the best so far.  The logarithm in its fast form is off by far less
// than the slack; the exact score is only taken of those that come that near to
// the warp's best, `mark` (a thread's own best is passed by some lane at almost
// every step).
template <typename T, typename F>
OSSM_DEV void race(const float* l, const float* e, int i, int n, float low, F stays, float inv_t, Best& b,
                   float& mark) {
  const float bar = mark - 1e-4f;
  uint32_t near = 0;
#pragma unroll
  for (int k = 0; k < Vec<T>::n; ++k) {
    const float x = l[k] * inv_t, s = fmaf(-0.693147181f, lg2(e[k]), fmaf(1e-6f, fabsf(x), x));
    near |= k < n && l[k] >= low && !(s < bar) ? 1u << k : 0u;
  }
  if (near) {
#pragma unroll
    for (int k = 0; k < Vec<T>::n; ++k)
      if ((near >> k & 1u) && stays(l[k], i + k)) better(b, score_of(l[k], inv_t, e[k]), i + k);
  }
  mark = logit_of((u64)__reduce_max_sync(~0u, ord(b.i < 0 ? -INFINITY : b.s)) << 32);
}

// What the CTAs of a cluster tell each other.
struct Told {
  float m, z;      // largest logit; sum of the weights relative to it, in fp32
  u64 whole;       // the row's mass (the first CTA's)
  uint32_t tk;     // order bits that at least top_k candidates reach
  float guess;     // where its part of the tail begins
  int count;       // candidates collected (the first CTA's)
  Best best;
};

// A row without filters: the best score of all its candidates.
template <int NT, typename T>
OSSM_DEV void open_row(const T* lg, const float* nz, int V, float inv_t, int rank, int nrank, Best* bests, Told& told,
                       int64_t* out) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  Best b{0.f, -1};
  float mark = -INFINITY;
  scan_noise<NT>(lg, nz, V, rank, nrank, [&](const float* l, const float* e, int i, int n) {
    race<T>(l, e, i, n, kLowest, [](float, int) { return true; }, inv_t, b, mark);
  });
  b = block_best<NT>(b, bests);
  if (nrank > 1) {
    if (tid == 0) told.best = b;
    cluster.sync();
    if (rank == 0 && tid < 32) {
      b = Best{0.f, -1};
      if (tid < nrank) b = cluster.map_shared_rank(&told, tid)->best;
      for (int w = 16; w; w >>= 1) better(b, __shfl_xor_sync(~0u, b.s, w), __shfl_xor_sync(~0u, b.i, w));
    }
    cluster.sync();  // the others' memory is read before they leave
  }
  if (rank == 0 && tid == 0) *out = b.i;
}

// Every row without filters (known on the host).  Two CTAs of 512 threads an SM
// cover one another's loads and tails: 256 rows of 32000 fp32, 11.6 us back to
// back (10.0 us of reads; 15.1 us with one CTA of 1024; 14.4 us as a call among
// others), 256 of 131072 bf16, 33.5 us (30.8 of reads).  At 40 registers a
// thread the loads ahead spill (17 and 38 us).
template <typename T>
__global__ void __launch_bounds__(kOpen, 2) open_kernel(const Params p) {
  __shared__ Best bests[kOpen / 32];
  __shared__ Told told;
  const int nrank = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
  const i64 row = blockIdx.x / nrank;
  open_row<kOpen>(static_cast<const T*>(p.logits) + row * p.lst, p.noise + row * p.nst, p.V, p.inv_t, rank, nrank,
                  bests, told, p.out + row);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const Params p) {
  extern __shared__ u64 dynamic[];
  Room& room = *reinterpret_cast<Room*>(dynamic);
  __shared__ float redf[32];
  __shared__ Best bests[32];
  __shared__ Told told;
  cg::cluster_group cluster = cg::this_cluster();
  const int nrank = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / nrank, tid = threadIdx.x;
  const T* lg = static_cast<const T*>(p.logits) + row * p.lst;
  const float* nz = p.noise ? p.noise + row * p.nst : nullptr;
  const Row r = row_of(p, row);
  if (tid == 0) told.count = 0, told.whole = 0;

  if (r.open()) {
    open_row<kThreads>(lg, nz, p.V, r.inv_t, rank, nrank, bests, told, p.out + row);
    return;
  }

  // ---------------------------------------------------------------- the largest logit, the weights' sum
  const int top_k = r.greedy ? 1 : r.top_k;
  const bool by_mass = !r.greedy && r.top_p < 1.f;
  const bool need_z = by_mass && top_k == 0;
  const float c = fminf(r.inv_t * 1.44269504f, 3e38f);
  float m = -INFINITY, z = 0.f;
  scan(lg, p.V, rank, nrank, [&](const float* l, int, int n) {
    float top = l[0];
#pragma unroll
    for (int e = 1; e < Vec<T>::n; ++e)
      if (e < n) top = fmaxf(top, l[e]);
    if (top > m) {
      z = m == -INFINITY ? 0.f : z * ex2((m - top) * c);
      m = top;
    }
    if (need_z && live(m)) {
#pragma unroll
      for (int e = 0; e < Vec<T>::n; ++e)
        if (e < n) z += ex2((l[e] - m) * c);
    }
  });
  const float cta_m = block_reduce(m, redf, [](float a, float b) { return fmaxf(a, b); });
  if (need_z)
    z = block_reduce(live(m) ? z * (m == cta_m ? 1.f : ex2((m - cta_m) * c)) : 0.f, redf,
                     [](float a, float b) { return a + b; });
  // order bits that at least top_k of this CTA's threads' largest logits reach,
  // so at least top_k candidates: the 16 high bits by bisection
  uint32_t tk = 0;
  if (top_k && top_k <= kThreads) {
    const uint32_t mine = live(m) ? ord(m) : 0u;
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t t = tk | (1u << bit);
      if (__syncthreads_count(mine >= t) >= top_k) tk = t;
    }
  }
  if (nrank > 1) {
    if (tid == 0) {
      told.m = cta_m;
      told.z = z;
      told.tk = tk;
    }
    cluster.sync();
    // a lane for each of the others, in every warp
    const int lane = tid & 31;
    const Told* o = cluster.map_shared_rank(&told, min(lane, nrank - 1));
    const float om = o->m, oz = o->z;
    m = om;
    tk = __reduce_max_sync(~0u, o->tk);
#pragma unroll
    for (int w = 4; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, w));
    m = __shfl_sync(~0u, m, 0);
    z = need_z && lane < nrank && live(om) ? oz * (om == m ? 1.f : ex2((om - m) * c)) : 0.f;
#pragma unroll
    for (int w = 4; w; w >>= 1) z += __shfl_xor_sync(~0u, z, w);
    z = __shfl_sync(~0u, z, 0);
  } else {
    m = cta_m;
    __syncthreads();  // told.count is 0
  }
  if (!live(m)) {
    if (nrank > 1) cluster.sync();
    if (rank == 0 && tid == 0) p.out[row] = -1;
    return;
  }
  const Masses ms(m, r.inv_t);

  // ---------------------------------------------------------------- Bound, and the candidates above it
  // With top_k: its own bound alone, as its mass counts for top_p.  Without:
  // the candidates below (1 - top_p) z / V weigh less than (1 - top_p) z
  // together, so the prefix ends above them.  min_p only ever shortens.  The
  // logarithms' and the products' roundings are covered by the slack.
  uint32_t bound = tk;
  float lb = -INFINITY;  // the same as a logit, of the bounds by mass
  bool guessed = need_z && p.V / nrank >= kGuess;
  if (!(top_k && by_mass)) {
    float y = -INFINITY;
    if (need_z) y = logf((1.f - r.top_p) * z / (float)p.V);
    if (!r.greedy && r.min_p > 0.f) {
      const float by_min = logf(fminf(r.min_p, 1.f));
      guessed = guessed && by_min < y + 2.f;
      y = fmaxf(y, by_min);
    }
    if (y > -INFINITY && m < INFINITY) {
      lb = m + (y - 1e-3f - 1e-5f * fabsf(y)) / r.inv_t;
      lb = fminf(lb - 1e-5f * (fabsf(m) + fabsf(lb)), m);
      bound = max(bound, ord(lb));
    }
  }
  // That bound by mass leaves many more than the prefix in wide rows (30000 of
  // 131072 where it holds 4000).  A guess leaves fewer; whether the prefix ends
  // above it shows in the mass collected.  top-p 0.9, with and without: 1 x 32000
  // (4 CTAs) 21 and 26 us, 64 x 50257 28 and 38 us, 128 x 32000 24 and 28 us.
  // Where min_p's bound is the higher one by far it leaves few anyhow.  Up to a
  // factor of e^2: 128 rows with top-p and a small min-p of their own, V = 131072,
  // 52 to 63 us over three inputs, only where it is the lower one 52 to 100 us (V =
  // 50257: 27 and 30 us); up to e^4, where prefixes end below it and the row is
  // gone over, 43 us (50257).
  guessed = guessed && lb > -INFINITY && lb < m;
  if (guessed) {
    float g = guess_bound(lg, p.V, rank, nrank, m, lb, c, (1.f - r.top_p) * z / (float)nrank, room);
    if (nrank > 1) {  // the lowest of the CTAs'
      if (tid == 0) told.guess = g;
      cluster.sync();
      g = cluster.map_shared_rank(&told, min(tid & 31, nrank - 1))->guess;
#pragma unroll
      for (int w = 16; w; w >>= 1) g = fminf(g, __shfl_xor_sync(~0u, g, w));
    }
    guessed = g > lb;
    bound = max(bound, ord(g));
  }
  Told* first = nrank > 1 ? cluster.map_shared_rank(&told, 0) : &told;
  u64* first_list = nrank > 1 ? cluster.map_shared_rank(room.list, 0) : room.list;
  const float low = bound ? fmaxf(logit_of((u64)bound << 32), kLowest) : kLowest;
  // next to an infinite logit nothing else has weight; the sum is taken over the candidates then
  const bool sum = need_z && m < INFINITY;
  u64 whole;
  if (!sum) {
    collect<false>(lg, p.V, rank, nrank, low, ms, &first->count, first_list);
  } else {
    whole = collect<true>(lg, p.V, rank, nrank, low, ms, &first->count, first_list);
#pragma unroll
    for (int w = 16; w; w >>= 1) whole += __shfl_xor_sync(~0u, whole, w);
    if ((tid & 31) == 0) add64(&first->whole, whole);
  }
  if (nrank > 1)
    cluster.sync();
  else
    __syncthreads();
  if (rank != 0) return;

  // ---------------------------------------------------------------- the prefix and its best score
  const int N = told.count;
  whole = told.whole;
  Best b{0.f, -1};
  u64 keep = 0;  // the prefix's last key
  bool by_list = N <= kList;
  if (by_list && r.greedy) {
    for (int e = tid; e < N; e += kThreads) keep = max(keep, room.list[e]);
    keep = block_reduce(keep, room.red, [](u64 a, u64 b) { return max(a, b); });
  } else if (by_list) {
    const u64 target = whole ? share(r.top_p, whole) : 0;
    if (N <= kRank && (top_k || by_mass)) {
      order(room.list, N);
      int n = top_k ? min(top_k, N) : N;
      if (by_mass) {
        const int stay = reaching(room.list, n, ms, r, target, room.red);
        by_list = !(guessed && stay > n);
        n = min(n, stay);
      }
      if (n) keep = room.list[n - 1];
    } else {
      if (top_k && top_k < N) keep = select_list(r, N, ms, 0, top_k, 0, room);
      if (by_mass) keep = select_list(r, N, ms, keep, 0, target, room);
      by_list = !(guessed && keep == 0);  // 0: the guess was too high
    }
  }
  if (by_list && r.greedy) {
    if (tid == 0) better(b, 0.f, index_of(keep));
  } else if (by_list) {
    constexpr int U = 4;  // noises on their way at a time
    for (int e = tid; e < N; e += U * kThreads) {
      u64 key[U];
      float x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        key[k] = e + k * kThreads < N ? room.list[e + k * kThreads] : 0;
        if (key[k] < keep || (r.min_p > 0.f && weight(logit_of(key[k]), m, r.inv_t) < r.min_p)) key[k] = 0;
        if (key[k]) x[k] = nz[index_of(key[k])];
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (key[k]) better(b, score_of(logit_of(key[k]), r.inv_t, x[k]), index_of(key[k]));
    }
  } else {
    if (!r.greedy && tid == 0) {  // the last pass reads the noise: on its way to L2 meanwhile
      const uintptr_t a = ((uintptr_t)nz + 15) & ~(uintptr_t)15, z = (uintptr_t)(nz + p.V) & ~(uintptr_t)15;
      for (uintptr_t x = a; x < z; x += 32768)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(x), "r"((uint32_t)min((u64)32768, (u64)(z - x)))
                     : "memory");
    }
    u64 top = 0;
    keep = 0;
    float least = INFINITY;
    if (r.greedy || top_k || !live(lb)) {
      scan(lg, p.V, 0, 1, [&](const float* l, int i, int n) {
#pragma unroll
        for (int e = 0; e < Vec<T>::n; ++e)
          if (e < n && live(l[e])) top = max(top, key_of(l[e], i + e)), least = fminf(least, l[e]);
      });
      top = block_reduce(top, room.red, [](u64 a, u64 b) { return max(a, b); });
      least = block_reduce(least, redf, [](float a, float b) { return fminf(a, b); });
    }
    if (r.greedy) {
      keep = top;
    } else {
      if (top_k) keep = select_row(r, lg, p.V, ms, least, 0, top_k, 0, room);
      if (by_mass)
        keep = select_row(r, lg, p.V, ms, live(lb) ? lb : top_k ? logit_of(keep) : least, keep, 0, whole, room);
    }
    const float end = keep ? logit_of(keep) : -INFINITY;  // the last one's logit: only there the index decides
    if (r.greedy) {
      if (tid == 0) better(b, 0.f, index_of(keep));
    } else {
      float mark = -INFINITY;
      auto stays = [&](float l, int i) {
        const u64 key = key_of(l, i);
        return key >= keep && (!(r.min_p > 0.f) || weight(l, m, r.inv_t) >= r.min_p);
      };
      scan_noise<kThreads>(lg, nz, p.V, 0, 1, [&](const float* l, const float* e, int i, int n) {
        race<T>(l, e, i, n, fmaxf(fmaxf(end, lb), kLowest), stays, r.inv_t, b, mark);
      });
    }
  }
  b = block_best<kThreads>(b, bests);
  if (tid == 0) p.out[row] = b.i;
}

// CTAs a row: as many as fill the GPU about once, with 4096 logits each at
// least.  One row of 32000 with top-k 50 took 10.4 us with 4 CTAs and 13.7 us
// with 8 (the bound, of each CTA's own threads, gets weak: 377 candidates are
// collected instead of 90), 10.7 us with one.
template <typename T>
cudaError_t launch(const Params& p, int B, cudaStream_t st) {
  const int sms = device_sms();
  const bool open = p.noise && !p.t_row && !p.k_row && !p.p_row && !p.m_row && p.inv_t > 0.f && p.inv_t < INFINITY &&
                    (p.top_k <= 0 || p.top_k >= p.V) && p.top_p >= 1.f && !(p.min_p > 0.f);
  int c = 1;
  while (c < 8 && (i64)B * c * (open ? 1 : 2) <= sms && p.V / (2 * c) >= 4096) c *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)B * c);
  cfg.blockDim = dim3(open ? kOpen : kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = c, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (open) return cudaLaunchKernelEx(&cfg, open_kernel<T>, p);
  cfg.dynamicSmemBytes = sizeof(Room);
  const cudaError_t e =
      cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Room));
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
}

}  // namespace smp
}  // namespace ossm

using namespace ossm;

extern "C" int ossm_sample_tokens(const ossm_sample_args* a, ossm_stream_t stream) {
  if (!a || a->B < 0 || a->B > (1 << 27) || a->V < 1 || a->V >= (1 << 23) || !a->logits || !a->out) return OSSM_EINVAL;
  const int el = a->dtype == OSSM_F32 ? 4 : 2;
  if ((a->dtype != OSSM_F32 && a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) || (uintptr_t)a->logits % el ||
      (uintptr_t)a->noise % 4 || (uintptr_t)a->out % 8)
    return OSSM_EINVAL;
  if (!(a->top_p >= 0.f) || !(a->min_p >= 0.f) || a->top_k < 0 || !(a->inv_temperature >= 0.f)) return OSSM_EINVAL;
  if (a->B == 0) return OSSM_OK;
  const smp::Params p{a->V, a->logits, a->logits_stride, a->noise, a->noise_stride, a->inv_temperature, a->top_p,
                      a->min_p, a->top_k, a->temperature_row, a->top_p_row, a->min_p_row, a->top_k_row, a->out};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == OSSM_F32)
    e = smp::launch<float>(p, a->B, st);
  else if (a->dtype == OSSM_BF16)
    e = smp::launch<__nv_bfloat16>(p, a->B, st);
  else
    e = smp::launch<__half>(p, a->B, st);
  return e == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}
