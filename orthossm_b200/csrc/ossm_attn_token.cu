// Attention of few queries a sequence against a long cache: single tokens,
// short pieces of prompts.
//
// Bound by the read of K and V, once each; the products run on mma.sync, whose
// rate is far above what the reads can feed.  A work item is 16 query rows that
// share their keys (row = query * heads per key head + head of the group) and
// the keys they see.  Warps work alone: each takes 16 keys at a time through a
// ring of its own (cp.async), with its own running maximum, sums and output;
// the four warps of a CTA add up at the end of a piece.
//
// As for prompts, the items of all sequences form one line that is cut evenly
// over the CTAs, whatever the lengths; partial results meet in the workspace,
// joined in the order of the cut by whichever CTA finishes the item last.
//
// The weights enter the product with V as a sum of two 16-bit terms, so that
// their rounding does not add to the output's; the reads hide that product.
//
// Measured as calls among others: 64 streams of up to 8192 keys, 32/8 heads of
// 128: 189 us, 6.4 TB/s (0.98 of measured copy bandwidth); one stream of 1048576
// keys, 8 heads of 64: 359 to 378 us, 6.0 to 5.7 TB/s on different GPUs; 32
// streams with a window of 512: 14.4 us (5.1 us of reads: bound by the launch, the
// schedule and one item's chain of loads and merge).
#include <algorithm>

#include "ossm_attn.cuh"
#include "ossm_sm100.cuh"

namespace ossm {
namespace attn {
namespace tok {

using sm100::smem_u32;
typedef long long i64;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRows = 16;             // query rows of an item
constexpr int kWK = 16;               // keys of a warp's step
constexpr int kGroups = 256;          // entries of the line's prefix in shared memory
constexpr int kItemCost = 2;          // an item's start and end, in steps
constexpr int kMinPiece = 4;          // no cut closer to an item's edge
constexpr int kMinWork = 8;           // a CTA for each part of this length at most, and for each item
constexpr int kPairFrom = 32;         // steps a CTA from which items take two heads
constexpr int kJoin = 16;             // partial results joined at once
constexpr int kSecond = 2 * kMaxCtas;  // the second step's counters, one a CTA, follow those of the first

template <int HDP>
struct Cfg {
  static constexpr int kStages = HDP == 64 ? 4 : 3;
  static constexpr int kCtas = HDP == 64 ? 3 : 2;             // resident CTAs an SM
  static constexpr int kTile = kWK * HDP * 2;                 // bytes of a warp's K or V tile
  static constexpr int kSmem = kWarps * kStages * 2 * kTile;  // also holds the warps' outputs at the end
  static constexpr int kHeads = HDP == 64 ? 2 : 1;            // key heads of an item, at most
  static constexpr int kPart = kHeads * kRows;                // rows of a partial result
  static constexpr size_t kPartFloats = kPart * (HDP + 2);
  static_assert(kMaxSms * kCtas <= kMaxCtas && kSecond + kMaxCtas <= kCounters, "a counter of its own for each");
  static_assert(kSmem >= kWarps * kRows * HDP * 4, "outputs of the warps");
};

// An item takes `hp` neighbouring key heads, a warp one of them: with 64
// channels one head's row is 128 bytes, and reading the heads of a token far
// apart in time cost a sixth of the bandwidth (1048576 keys, 8 heads: 392 us,
// head-major 340 us).
struct Line {
  const Params& p;
  int hp;
  const i64* pre;
  int ngroups, gsz;
  Cuts<kMinPiece, kItemCost> cuts;

  struct Item {
    Seq q;
    int rb, kvh, n;  // row block, first key head, steps
    i64 start;
    OSSM_DEV i64 end() const { return start + n + kItemCost; }
  };
  // First key that some query sees, and one past the last.
  static OSSM_DEV int first_key(const Params& p, const Seq& q) {
    return p.window ? max(0, q.nk - q.nq - p.window + 1) : 0;
  }
  OSSM_DEV int chunk() const { return kWarps * kWK / hp; }  // keys of a CTA's step, the line's unit
  OSSM_DEV int steps(const Seq& q) const { return max(1, (q.nk - first_key(p, q) + chunk() - 1) / chunk()); }
  OSSM_DEV int blocks(const Seq& q) const {  // row blocks times groups of key heads
    return (int)(((i64)q.nq * (p.H / p.Hkv) + kRows - 1) / kRows) * (p.Hkv / hp);
  }
  OSSM_DEV Item at(i64 pos) const {
    int lo = 0, hi = ngroups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= pos) lo = mid; else hi = mid;
    }
    i64 base = pre[lo];
    Item it;
    for (int b = lo * gsz;; ++b) {
      it.q = seq_of(p, b);
      it.n = steps(it.q);
      const i64 len = (i64)blocks(it.q) * (it.n + kItemCost);
      if (pos < base + len || b + 1 >= min(p.B, (lo + 1) * gsz)) break;
      base += len;
    }
    const int u = (int)((pos - base) / (it.n + kItemCost));
    it.rb = u / (p.Hkv / hp);
    it.kvh = u % (p.Hkv / hp) * hp;
    it.start = base + (i64)u * (it.n + kItemCost);
    return it;
  }
  // Where CTA c's part begins (and the item there, if it is not past the item's end).
  OSSM_DEV i64 cut(int c, Item& it, bool& in) const {
    in = false;
    if (c >= cuts.ncta) return cuts.total;
    const i64 pos = c <= 0 ? 0 : cuts.place(c);
    it = at(pos);
    const i64 to = cuts.moved(pos, it.start, it.end());
    in = to < it.end();
    return to;
  }
  OSSM_DEV i64 cut(int c) const {
    Item it;
    bool in;
    return cut(c, it, in);
  }
};

template <typename T>
OSSM_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OSSM_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
OSSM_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
OSSM_DEV void cp16(uint32_t dst, const void* src, bool full) {  // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
// p0, p1 as the sum of two packed pairs.
template <typename T>
OSSM_DEV void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(p0, p1);
  const float2 h = to_f2<T>(hi);
  lo = pack2<T>(p0 - h.x, p1 - h.y);
}

// Byte offset of 16-byte chunk c of row r in a tile: rows of HDP channels, the
// chunks of 8 rows spread over the banks.
template <int HDP>
OSSM_DEV uint32_t off16(int r, int c) {
  return r * (HDP * 2) + ((c ^ (r & 7)) << 4);
}

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, Cfg<HDP>::kCtas) attn_token_kernel(const __grid_constant__ Params p) {
  using C = Cfg<HDP>;
  constexpr int CH = HDP / 8, KS = HDP / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ i64 pre[kGroups + 1];
  __shared__ unsigned long long n_items;
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  __shared__ float sm_p[kWarps][kRows][kWK];
  __shared__ int last_in;
  __shared__ i64 cuts[2];
  __shared__ Line::Item item;  // the first one, if item_in
  __shared__ bool item_in;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
  const int G = p.H / p.Hkv;
  const int gsz = (p.B + kGroups - 1) / kGroups, ngroups = (p.B + gsz - 1) / gsz;
  // One head an item; two where the line is long for the GPU, as they halve the
  // items (32 streams with a window of 512: 14 us with one, 23 us with two).
  Line ln{p, 1, pre, ngroups, gsz, {0, 0}};
  for (;;) {
    if (threadIdx.x == 0) n_items = 0;
    __syncthreads();
    unsigned long long mine = 0;
    for (int g = threadIdx.x; g < ngroups; g += kThreads) {
      i64 len = 0;
      for (int b = g * gsz; b < min(p.B, (g + 1) * gsz); ++b) {
        const Seq q = seq_of(p, b);
        const int nb = ln.blocks(q);
        len += (i64)nb * (ln.steps(q) + kItemCost);
        mine += nb;
      }
      pre[g + 1] = len;
    }
    mine = warp_sum(mine);
    if (lane == 0 && mine) atomicAdd(&n_items, mine);
    __syncthreads();
    if (warp == 0) {
      i64 run = 0;
      for (int g0 = 0; g0 < ngroups; g0 += 32) {
        i64 v = g0 + lane < ngroups ? pre[g0 + lane + 1] : 0;
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
          const i64 u = __shfl_up_sync(~0u, v, w);
          if (lane >= w) v += u;
        }
        if (g0 + lane < ngroups) pre[g0 + lane + 1] = run + v;
        run += __shfl_sync(~0u, v, 31);
      }
      if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
    ln.cuts.total = pre[ngroups];
    if (C::kHeads == 1 || ln.hp == 2 || p.Hkv % 2 || ln.cuts.total < (i64)kPairFrom * gridDim.x) break;
    ln.hp = 2;
    __syncthreads();
  }
  const int hp = ln.hp, sub = warp & (hp - 1), kw = warp / hp, nkw = kWarps / hp;  // head, place among its warps
  // twice the items: each item's edge is the nearest one to some cut, and short items get a CTA each
  ln.cuts.ncta = (int)min((i64)gridDim.x, max(2 * (i64)n_items, ln.cuts.total / kMinWork));
  if (cta >= ln.cuts.ncta) return;
  if (lane == 0 && warp < 2) {
    Line::Item it;
    bool in;
    cuts[warp] = ln.cut(cta + warp, it, in);
    if (warp == 0) {
      item = it;
      item_in = in;
    }
  }
  __syncthreads();
  bool known = item_in;

  const uint32_t ring = smem_u32(smem) + warp * (C::kStages * 2 * C::kTile);
  const uint8_t* ringp = smem + warp * (C::kStages * 2 * C::kTile);
  const int r4 = lane >> 2, c4 = lane & 3;  // this lane's rows r4, r4 + 8 and column pair in the fragments
  i64 pos = cuts[0];
  const i64 end = cuts[1];
  while (pos < end) {
    const Line::Item x = known ? item : ln.at(pos);
    known = false;
    const int a = (int)min(pos - x.start, (i64)x.n), b = (int)min(end - x.start, (i64)x.n);
    const bool head = pos == x.start;
    pos = min(end, x.end());
    if (a >= b) continue;
    const int off = x.q.nk - x.q.nq, lo = Line::first_key(p, x.q);
    const int kvh = x.kvh + sub;
    const int row0 = x.rb * kRows, nrows = (int)min((i64)kRows, (i64)x.q.nq * G - row0);
    const int i_first = row0 / G, i_last = (row0 + nrows - 1) / G;
    // the piece's keys that some row sees: the item's are those of the whole
    // sequence, whose other queries begin earlier or end later
    const int kbeg = max(lo + a * ln.chunk(), p.window ? i_first + off - p.window + 1 : 0);
    const int kend = min(min(x.q.nk, lo + b * ln.chunk()), i_last + off + 1);
    // positions of this lane's rows (rows past the block repeat its last)
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) at[h] = (row0 + min(r4 + 8 * h, nrows - 1)) / G + off;

    float o[HDP / 8][4];
#pragma unroll
    for (int i = 0; i < HDP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // this warp's tiles: kbeg + (kw + nkw u) * 16
    const int nt = kend > kbeg ? ((kend - kbeg + kWK - 1) / kWK - kw + nkw - 1) / nkw : 0;
    constexpr int RP = 32 / CH;  // rows a warp copies at once
    const int cr = lane / CH, cc = lane % CH;
    const T* kg = static_cast<const T*>(p.k) + (i64)x.q.k0 * p.kst + (i64)kvh * p.ksh + cc * 8;
    const T* vg = static_cast<const T*>(p.v) + (i64)x.q.k0 * p.vst + (i64)kvh * p.vsh + cc * 8;
    auto load = [&](int u) {
      if (u < nt) {
        const int key = kbeg + (kw + nkw * u) * kWK + cr;
        const uint32_t kd = ring + (u % C::kStages) * (2 * C::kTile), vd = kd + C::kTile;
        const T *ks = kg + (i64)key * p.kst, *vs = vg + (i64)key * p.vst;
#pragma unroll
        for (int i = 0; i < kWK / RP; ++i) {
          const bool in = key + i * RP < kend && cc * 8 < p.hd;
          cp16(kd + off16<HDP>(cr + i * RP, cc), in ? ks + (i64)(i * RP) * p.kst : static_cast<const T*>(p.k), in);
          cp16(vd + off16<HDP>(cr + i * RP, cc), in ? vs + (i64)(i * RP) * p.vst : static_cast<const T*>(p.v), in);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int u = 0; u < C::kStages - 1; ++u) load(u);
    // Q fragments
    uint32_t qf[KS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r4 + 8 * h, i = (row0 + r) / G, hd_ = kvh * G + (row0 + r) % G;
      const T* q = static_cast<const T*>(p.q) + (i64)(x.q.q0 + i) * p.qst + (i64)hd_ * p.qsh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = ks * 16 + e * 8 + c4 * 2;
          qf[ks][h + 2 * e] = r < nrows && d < p.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
    }
    for (int u = 0; u < nt; ++u) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
      __syncwarp();
      load(u + C::kStages - 1);
      const uint32_t kd = ring + (u % C::kStages) * (2 * C::kTile), vd = kd + C::kTile;
      const int key0 = kbeg + (kw + nkw * u) * kWK;
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t f[4];  // keys 0-7: f0 f1; keys 8-15: f2 f3
        ldsm4(f, kd + off16<HDP>((lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)));
        mma16816<T>(s[0], qf[ks], f[0], f[1]);
        mma16816<T>(s[1], qf[ks], f[2], f[3]);
      }
      // some row does not see the whole tile, or it reaches past the piece
      const bool part = key0 + kWK - 1 > i_first + off || key0 + kWK > kend ||
                        (p.window && key0 <= i_last + off - p.window);
      uint32_t seen = 0xffu;  // bit 4 h + 2 nb + e: row r4 + 8 h, key 8 nb + 2 c4 + e
      if (part) {
        seen = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = key0 + 8 * nb + 2 * c4 + e;
              if (key <= at[h] && !(p.window && key <= at[h] - p.window) && key < kend)
                seen |= 1u << (4 * h + 2 * nb + e);
              else
                s[nb][2 * h + e] = -INFINITY;
            }
      }
      // maximum: as long as no row has grown by more than 2^8 since the
      // exponents' last maximum, that one stays
      float top[2];
      bool grow = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1])) * p.scale2;
        grow |= top[h] > m[h] + 8.f;
      }
      if (__any_sync(~0u, grow)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 2));
          const float mn = top[h] > m[h] + 8.f ? top[h] : m[h];
          const float f = mn == m[h] ? 1.f : ex2(m[h] - mn);
          m[h] = mn;
          l[h] *= f;
#pragma unroll
          for (int i = 0; i < HDP / 8; ++i) {
            o[i][2 * h] *= f;
            o[i][2 * h + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float ms = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[nb][2 * h + e] = ex2(fmaf(s[nb][2 * h + e], p.scale2, -ms));
            l[h] += s[nb][2 * h + e];
          }
      }
      // A weight of 0 times a non-finite value is NaN.  Keys outside [kbeg, kend),
      // which no row sees, were loaded as zeros; where rows see different keys of
      // the tile and one of its values is not finite, the product is taken key by
      // key.  Rows of one query all see every key loaded.
      bool bad = false;
      if (part && i_first != i_last) {
        const uint8_t* vt = ringp + (u % C::kStages) * (2 * C::kTile) + C::kTile;
        for (int i = lane; i < kWK * CH; i += 32) {
          const uint4 w = *reinterpret_cast<const uint4*>(vt + i * 16);
          bad |= nonfinite2<T>(w.x) || nonfinite2<T>(w.y) || nonfinite2<T>(w.z) || nonfinite2<T>(w.w);
        }
        bad = __any_sync(~0u, bad);
        if (bad) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
              for (int e = 0; e < 2; ++e)  // hidden keys are marked by a negative weight
                sm_p[warp][r4 + 8 * h][8 * nb + 2 * c4 + e] =
                    (seen >> (4 * h + 2 * nb + e) & 1u) ? s[nb][2 * h + e] : -1.f;
          __syncwarp();
          for (int k = 0; k < kWK; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float w = sm_p[warp][r4 + 8 * h][k];
              if (w < 0.f) continue;
#pragma unroll
              for (int i = 0; i < HDP / 8; ++i) {
                const float2 v2 = to_f2<T>(*reinterpret_cast<const uint32_t*>(vt + off16<HDP>(k, i) + c4 * 4));
                o[i][2 * h] = fmaf(w, v2.x, o[i][2 * h]);
                o[i][2 * h + 1] = fmaf(w, v2.y, o[i][2 * h + 1]);
              }
            }
          }
          __syncwarp();
        }
      }
      if (!bad) {
        uint32_t ph[4], pl[4];
        split2<T>(s[0][0], s[0][1], ph[0], pl[0]);
        split2<T>(s[0][2], s[0][3], ph[1], pl[1]);
        split2<T>(s[1][0], s[1][1], ph[2], pl[2]);
        split2<T>(s[1][2], s[1][3], ph[3], pl[3]);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t f[4];  // channels 16 i + 0-7: f0 f1; 8-15: f2 f3
          ldsm4t(f, vd + off16<HDP>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * i + (lane >> 4)));
          mma16816<T>(o[2 * i], ph, f[0], f[1]);
          mma16816<T>(o[2 * i], pl, f[0], f[1]);
          mma16816<T>(o[2 * i + 1], ph, f[2], f[3]);
          mma16816<T>(o[2 * i + 1], pl, f[2], f[3]);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // the warps' results side by side in the ring's memory
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(~0u, l[h], 1);
      l[h] += __shfl_xor_sync(~0u, l[h], 2);
    }
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);  // [warp][row][HDP]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r4 + 8 * h;
      if (c4 == 0) {
        sm_m[warp][r] = m[h];
        sm_l[warp][r] = l[h];
      }
      if (r < nrows) {
#pragma unroll
        for (int i = 0; i < HDP / 8; ++i)
          *reinterpret_cast<float2*>(so + (warp * kRows + r) * HDP + 8 * i + 2 * c4) =
              make_float2(o[i][2 * h], o[i][2 * h + 1]);
      }
    }
    __syncthreads();
    const bool split = b - a < x.n;
    const int first = split ? (head ? cta : ln.cuts.first_of(x.start, x.end())) : cta;
    auto slot = [&](int c) {  // of CTA c's piece of this item
      return p.part + (size_t)(c == first ? 2 * c + 1 : 2 * c) * C::kPartFloats;
    };
    float* part = slot(cta);
    T* out = static_cast<T*>(p.out);
    // rows of the item's heads one after the other
    auto out_at = [&](int rr) {
      const int h = rr / nrows, r = row0 + rr % nrows;
      return out + (i64)(x.q.q0 + r / G) * p.ost + (i64)((x.kvh + h) * G + r % G) * p.osh;
    };
    const int nout = nrows * hp * CH;
    for (int e = threadIdx.x; e < nout; e += kThreads) {
      const int rr = e / CH, r = rr % nrows, h = rr / nrows, d = (e % CH) * 8;
      float M = -INFINITY;
      for (int w = h; w < kWarps; w += hp) M = fmaxf(M, sm_m[w][r]);
      const float Ms = M == -INFINITY ? 0.f : M;
      float acc[8] = {}, L = 0.f;
      for (int w = h; w < kWarps; w += hp) {
        if (sm_m[w][r] == -INFINITY && sm_l[w][r] == 0.f) continue;  // a warp that has seen no key
        const float f = ex2(sm_m[w][r] - Ms);
        L += f * sm_l[w][r];
        const float* q = so + (w * kRows + r) * HDP + d;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(f, q[i], acc[i]);
      }
      if (split) {
        if (d == 0) {
          part[rr] = M;
          part[C::kPart + rr] = L;
        }
        float4* po = reinterpret_cast<float4*>(part + 2 * C::kPart + rr * HDP + d);
        po[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        po[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else if (d < p.hd) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint4*>(out_at(rr) + d) =
            make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                       pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv));
      }
    }
    if (split) {
      const int last = ln.cuts.last_of(x.start, x.end(), x.start + x.n - 1);
      // Is this the last of n arrivals at a counter?  Then the others' partial results are there to read.
      auto arrive = [&](uint32_t* count, int n) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          last_in = atomicAdd(count, 1u) == (uint32_t)n - 1;
          if (last_in) *count = 0;  // for the next call
        }
        __syncthreads();
        const bool r = last_in;
        __threadfence();
        return r;
      };
      // The sum of n partial results, to the output or in place of the first.
      auto join = [&](auto piece, int n, float* to) {
        for (int e0 = 0; e0 < nout; e0 += kThreads) {
          const int e = e0 + threadIdx.x, r = e / CH, d = (e % CH) * 8;
          float M = -INFINITY, L = 0.f, acc[8] = {};
          if (e < nout) {
            for (int k0 = 0; k0 < n; k0 += 8) {
              float pm[8], pl[8];
              float4 u[8], v[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                pm[k] = -INFINITY, pl[k] = 0.f;
                u[k] = v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k < n) {
                  const float* q = piece(k0 + k);
                  pm[k] = __ldcg(q + r);
                  pl[k] = __ldcg(q + C::kPart + r);
                  u[k] = __ldcg(reinterpret_cast<const float4*>(q + 2 * C::kPart + r * HDP + d));
                  v[k] = __ldcg(reinterpret_cast<const float4*>(q + 2 * C::kPart + r * HDP + d) + 1);
                }
              }
              float top = M;
#pragma unroll
              for (int k = 0; k < 8; ++k) top = fmaxf(top, pm[k]);
              const float ms = top == -INFINITY ? 0.f : top, f0 = ex2(M - ms);
              M = top;
              L *= f0;
#pragma unroll
              for (int i = 0; i < 8; ++i) acc[i] *= f0;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float f = ex2(pm[k] - ms);
                L = fmaf(f, pl[k], L);
                acc[0] = fmaf(f, u[k].x, acc[0]), acc[1] = fmaf(f, u[k].y, acc[1]);
                acc[2] = fmaf(f, u[k].z, acc[2]), acc[3] = fmaf(f, u[k].w, acc[3]);
                acc[4] = fmaf(f, v[k].x, acc[4]), acc[5] = fmaf(f, v[k].y, acc[5]);
                acc[6] = fmaf(f, v[k].z, acc[6]), acc[7] = fmaf(f, v[k].w, acc[7]);
              }
            }
          }
          __syncthreads();  // `to` is read by all before it is written
          if (e >= nout) continue;
          if (to) {
            if (d == 0) {
              to[r] = M;
              to[C::kPart + r] = L;
            }
            float4* po = reinterpret_cast<float4*>(to + 2 * C::kPart + r * HDP + d);
            po[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            po[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          } else if (d < p.hd) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            *reinterpret_cast<uint4*>(out_at(r) + d) =
                make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                           pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv));
          }
        }
      };
      // Many pieces are joined in two steps, groups of neighbouring CTAs first:
      // one CTA alone would read all of them at its own small share of L2.
      const int np = last - first + 1;
      if (np <= kJoin) {
        if (arrive(p.counts + kSecond + first, np))
          join([&](int k) { return slot(first + k); }, np, static_cast<float*>(nullptr));
      } else {
        const int g0 = max(first, cta / kJoin * kJoin), g1 = min(last, cta / kJoin * kJoin + kJoin - 1);
        const int ng = last / kJoin - first / kJoin + 1;
        if (arrive(p.counts + (g0 == first ? 2 * g0 + 1 : 2 * g0), g1 - g0 + 1)) {
          join([&](int k) { return slot(g0 + k); }, g1 - g0 + 1, slot(g0));
          if (arrive(p.counts + kSecond + first, ng))
            join([&](int k) { return slot(k ? (first / kJoin + k) * kJoin : first); }, ng,
                 static_cast<float*>(nullptr));
        }
      }
    }
    __syncthreads();  // the ring's memory is read before the next piece fills it
  }
}

template <typename T, int HDP>
cudaError_t launch(const Params& p, int sms, cudaStream_t st) {
  using C = Cfg<HDP>;
  auto kern = attn_token_kernel<T, HDP>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kern, C::kSmem, done);
  if (e != cudaSuccess) return e;
  kern<<<sms * C::kCtas, kThreads, C::kSmem, st>>>(p);
  return cudaGetLastError();
}

}  // namespace tok

// Floats of the partial results of one SM's CTAs, and how many CTAs that is.
size_t token_part_floats(int hd) {
  return hd <= 64 ? 2 * tok::Cfg<64>::kCtas * tok::Cfg<64>::kPartFloats
                  : 2 * tok::Cfg<128>::kCtas * tok::Cfg<128>::kPartFloats;
}

int token_forward(const ossm_attn_args* a, const Params& p, int sms, cudaStream_t st) {
  const bool bf = a->dtype == OSSM_BF16;
  cudaError_t e;
  if (p.hd <= 64)
    e = bf ? tok::launch<__nv_bfloat16, 64>(p, sms, st) : tok::launch<__half, 64>(p, sms, st);
  else
    e = bf ? tok::launch<__nv_bfloat16, 128>(p, sms, st) : tok::launch<__half, 128>(p, sms, st);
  return e == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

}  // namespace attn
}  // namespace ossm
