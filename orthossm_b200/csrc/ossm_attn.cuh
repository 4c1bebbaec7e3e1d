// What the attention kernels share: arguments, a sequence's rows, types.
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include <type_traits>

#include "orthossm_b200.h"
#include "ossm_common.cuh"

namespace ossm {
namespace attn {

constexpr int kMaxSeqs = 16384;
constexpr int kMaxHD = 128;
constexpr int kMaxSms = 256;             // SMs that are used, at most
constexpr int kMaxCtas = 4 * kMaxSms;    // of a kernel's grid, at most
constexpr int kCounters = 3 * kMaxCtas;  // two a CTA, then one a CTA (the token kernel's second step)
constexpr long long kMaxRows = 1LL << 30;  // positions and their differences stay within 32 bits

// Lets a kernel have `bytes` of dynamic shared memory, once a device.
template <typename K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

struct Params {
  int B, H, Hkv, hd;
  int Tq, Tk;
  const void *q, *k, *v;
  void* out;
  long long qst, qsh, kst, ksh, vst, vsh, ost, osh;
  const int *cu_q, *cu_k, *kv_len;
  int window;      // 0: none
  float scale2;    // scale * log2(e): the softmax runs on base-2 exponents
  WsHeader* hdr;
  uint32_t* counts;  // [kCounters] progress of the items that are cut (0 between calls)
  float* part;       // per CTA two partial results
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

// A line of work items of length `total`, cut into ncta parts.  A cut within
// `near` of its item's edge moves to the edge (never closer than kMinPiece to
// the start, or kMinPiece + kItemCost to the end).
template <int kMinPiece, int kItemCost>
struct Cuts {
  long long total;
  int ncta;
  OSSM_DEV long long place(int c) const {  // of cut c, before it moves
    return total / ncta * c + total % ncta * c / ncta;
  }
  OSSM_DEV long long moved(long long pos, long long start, long long end) const {  // of a cut in item [start, end)
    const long long near = max((long long)kMinPiece, total / ncta / 16);
    if (pos - start <= near && pos - start <= end - pos) return start;
    if (end - pos <= near + kItemCost) return end;
    return pos - start <= near ? start : pos;
  }
  // The CTA whose part holds the item's start: the last whose cut is there or before.
  OSSM_DEV int first_of(long long start, long long end) const {
    int c = min(ncta - 1, (int)((double)start * ncta / (double)total));
    while (c > 0 && place(c) > start) --c;
    for (; c + 1 < ncta; ++c) {
      const long long q = place(c + 1);
      if (q > start && (q >= end || moved(q, start, end) > start)) break;
    }
    return c;
  }
  // The CTA whose part holds the item's last step, at `last`.
  OSSM_DEV int last_of(long long start, long long end, long long last) const {
    int c = min(ncta - 1, (int)((double)end * ncta / (double)total));
    while (c > 0 && (place(c) >= end || (place(c) > start && moved(place(c), start, end) > last))) --c;
    for (; c + 1 < ncta; ++c) {
      const long long q = place(c + 1);
      if (q >= end || (q > start && moved(q, start, end) > last)) break;
    }
    return c;
  }
};

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
OSSM_DEV uint32_t pack2(float lo, float hi);
template <>
OSSM_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
OSSM_DEV uint32_t pack2<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
// An infinity or NaN in either half of a packed pair.
template <typename T>
OSSM_DEV bool nonfinite2(uint32_t u) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (u & e) == e || (u & (e << 16)) == (e << 16);
}

OSSM_DEV unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(~0u, v, w);
  return v;
}
OSSM_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
OSSM_DEV float ex2(float x) {  // 2^x, relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace attn
}  // namespace ossm
