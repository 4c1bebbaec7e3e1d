// Attention of many queries a sequence: prompts, pieces of prompts.
//
// Work item: two tiles of 128 rows that share their keys.  A row is a query of
// one of g heads (row = query * g + head), g a power of two that divides the
// heads per key head, so that a few queries of a large group still fill a
// tile.  An item walks its range of 128-key tiles once with a running maximum
// and sum per row.
//
// One persistent CTA per SM, three warpgroups:
//   warps 0-3, 4-7  softmax of tile 0 / 1: a thread owns a row.  Scores from
//                   tensor memory, mask, maximum, exponentials, weights to
//                   tensor memory; at the end the output row out of the
//                   accumulator.  They also look through the V tiles that some
//                   row does not see whole (hidden values, below).
//   warp 8          issues the products S_t = Q_t K^T (tcgen05.mma, both
//                   operands in shared memory).
//   warp 9          walks the schedule, loads Q, K and V tiles by TMA.
//   warps 10, 11    issue O_t += P_t V for tile 0 / 1 (P_t in tensor memory, V
//                   read MN-major, so it is never transposed).
// One warp for all products spent its time waiting (16384 causal, 16 heads of
// 128: 1157 us against 937 us with three).
// Tensor memory (512 columns): scores, weights P_0 P_1, accumulators O_0 O_1.
// Up to 64 channels each tile has a score buffer of its own; above that there
// is room for one, which the tiles use in turn: a softmax takes its scores
// into registers at once and frees the buffer, and the next ones are formed
// while it computes.
//
// The weights enter the product rounded to the inputs' 16 bits, as the tensor
// core takes them (their sum is of the fp32 values): outputs are 1.2 to 1.4 times
// as far from float64 as with fp32 weights (a window of 512, bf16: 2.2e-3 and
// 1.6e-3 of their norm; 16384 causal, fp16: 2.4e-4 and 1.9e-4).  As two 16-bit
// parts they would take the product with V twice, on the pipe that bounds it.
//
// The maximum that the exponents are taken against follows the true one only
// when a row has grown by more than 2^8 since: the weights then stay below
// 2^8 and the accumulator is rescaled in a few tiles of a row instead of all.
//
// Schedule: the items of all sequences in one line, an item as long as its
// number of key tiles plus kItemCost; the line is cut into equal parts, one a
// CTA, so that causal masks and ragged lengths balance whatever they are.  A
// cut near an item's edge moves to the edge; an item that stays cut leaves
// partial sums in the workspace, and whichever CTA finishes it last joins
// them, in the order of the cut.
//
// What bounds it: a step of an item (two tiles, 128 keys) is 1024 (64 channels)
// or 2048 cycles (128) of the tensor core and 2048 of the special function unit
// (16 exponentials a clock and SM); of the softmax's other work a part overlaps
// with the other tile's exponentials.  Measured in bursts of 10 calls: 16384
// causal, fp16, 16 heads of 128: 910 us, 1209 TFLOP/s (0.74 of measured cuBLAS;
// 886 us on another GPU; called for longer, at the power cap, 1026 to 1070 us,
// 0.78 to 0.75 of cuBLAS under it); 8 heads of 64: 376 us; 2 x 16384 with a
// window of 512, 8 heads of 64: 88 us; 3 x 4096, 32/8 heads of 128: 365 us.  64
// bytes a thread are spilled.  Tried and slower: part of the exponentials as a
// polynomial on the FMA pipe (1 to 3 pairs of 8: +3 to +11 %), the tiles taking
// turns at them (+3 to +13 %), a row on two threads (16 softmax warps: +25 % at
// 128 channels).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "ossm_attn.cuh"
#include "ossm_sm100.cuh"

namespace ossm {
namespace fast {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
}
namespace attn {

using namespace sm100;

constexpr int kT = 128;             // query rows and keys of a tile
constexpr int kThreads = 384;       // three warpgroups of 168 registers a thread at launch
constexpr int kGroups = 1024;       // entries of the schedule's prefix in shared memory
constexpr int kItemCost = 2;        // an item's start and end, in key tiles
constexpr int kMinPiece = 6;        // no cut closer to an item's edge
constexpr int kBox = kT * 128;      // bytes of a [128 rows x 64 channels] box

// ---------------------------------------------------------------- schedule
typedef long long i64;

// Positions are divided by powers of two only: shifts, rounding down.
constexpr int kLT = 7;  // log2 of a tile's rows and keys

// sum over i < n of max(0, floor((x + i 2^lq) / 128))
OSSM_DEV i64 ramp(int n, int x, int lq) {
  if (lq >= kLT) {  // floor(x / 128) + i s
    const int a = x >> kLT, ls = lq - kLT;
    const int i0 = a >= 0 ? 0 : (-a + (1 << ls) - 1) >> ls;
    const i64 c = max(0, n - i0);
    return c * a + ((c * i0 + c * (c - 1) / 2) << ls);
  }
  const int lr = kLT - lq;  // floor((floor(x / 2^lq) + i) / 2^lr)
  auto upto = [lr](i64 m) {
    const i64 t = m > 0 ? m >> lr : 0;
    return m > 0 ? ((t * (t - 1) / 2) << lr) + (m - (t << lr)) * t : 0;
  };
  const i64 c = x >> lq;
  return upto(c + n) - upto(c);
}

// A sequence's blocks of 2 * 128 rows, 2^lq queries each: block i walks key
// tiles [lo(i), hi(i)).
struct Shape {
  int nblk, lq, t;  // t: the sequence's key tiles
  int x_lo, x_hi;   // lo(i) = floor((x_lo + i 2^lq) / 128), hi(i) = floor((x_hi + i 2^lq) / 128), within 0 .. t
  OSSM_DEV int lo(int i) const { return max(0, (x_lo + (i << lq)) >> kLT); }
  OSSM_DEV int hi(int i) const { return min(max(0, (x_hi + (i << lq)) >> kLT), t); }
  OSSM_DEV i64 before(int i) const {  // length of the blocks before i
    return ramp(i, x_hi, lq) - ramp(i, x_hi - (t << kLT), lq) - ramp(i, x_lo, lq) + (i64)i * kItemCost;
  }
};
OSSM_DEV Shape shape_of(const Params& p, const Seq& s, int lg) {
  const int off = s.nk - s.nq;
  Shape f;
  f.lq = kLT + 1 - lg;
  f.nblk = (s.nq + (1 << f.lq) - 1) >> f.lq;
  f.t = (s.nk + kT - 1) >> kLT;
  f.x_hi = off + (1 << f.lq) + kT - 1;  // the keys up to the block's last query, in tiles, rounded up
  // no window: the lower edge stays at 0 for every block
  f.x_lo = p.window ? off - p.window + 1 : -(f.nblk << f.lq);
  return f;
}

struct Sched {
  const Params& p;
  const i64* pre;  // [ngroups + 1] length of the line before each group of sequences
  int ngroups, gsz, lg, units;
  Cuts<kMinPiece, kItemCost> cuts;

  struct Item {
    Seq q;
    Shape f;
    int unit, blk;
    i64 start;  // on the line
    OSSM_DEV int n() const { return f.hi(blk) - f.lo(blk); }
    OSSM_DEV i64 end() const { return start + n() + kItemCost; }
  };

  // The item at a position of the line (0 <= pos < total).
  OSSM_DEV Item at(i64 pos) const {
    int lo = 0, hi = ngroups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= pos) lo = mid; else hi = mid;
    }
    i64 base = pre[lo];
    Item it;
    i64 one = 0;
    for (int b = lo * gsz;; ++b) {
      it.q = seq_of(p, b);
      it.f = shape_of(p, it.q, lg);
      one = it.f.before(it.f.nblk);
      if (pos < base + one * units || b + 1 >= min(p.B, (lo + 1) * gsz)) break;
      base += one * units;
    }
    it.unit = (int)((pos - base) / one);
    base += it.unit * one;
    const i64 rel = pos - base;
    lo = 0, hi = it.f.nblk;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (it.f.before(mid) <= rel) lo = mid; else hi = mid;
    }
    it.blk = lo;
    it.start = base + it.f.before(lo);
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

// A CTA's share of one item, as the roles read it.
struct Piece {
  int live;                // 0: no more pieces
  int q0, off, k0, nk;     // the sequence
  int nrows;               // its rows
  int head, row0;          // first head; first row of tile 0 (tile 1: 128 further)
  int j0, j1;              // the piece's key tiles
  int lo[2], hi[2];        // each tile's share of them
  int w0[2], w1[2];        // key tiles that every row of the tile sees whole
  int split;               // the item has other pieces
  int slot, first, len;    // split: this piece's slot, the CTA with the item's first piece, the item's key tiles
  i64 start;               // split: the item's start on the line
};

constexpr int kPieces = 4;  // ring of pieces
struct Bars {
  uint64_t q_full[2], q_empty[2], s_full[2], s_free[2], p_ready[2], pv_done[2];
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
};

template <int HDP>
struct Cfg {
  static constexpr int kBoxes = HDP / 64;
  static constexpr int kTile = kBoxes * kBox;
  static constexpr int kSlots = HDP == 64 ? 4 : 2;  // ring slots of K, and of V
  static constexpr size_t kSmem = (2 + 2 * kSlots) * (size_t)kTile + 1024;
  // columns: scores of 128 keys (one buffer a tile, or one for both), weights
  // as pairs of 16 bits, accumulators
  static constexpr int kS = HDP == 64 ? 2 : 1;
  static constexpr uint32_t kCols = 512, kP = kS * kT, kO = kP + 2 * (kT / 2);
  static_assert(kO + 2 * HDP <= kCols, "tensor memory");
  static constexpr size_t kPartFloats = 2 * kT * (size_t)(HDP + 2);
};

// Instruction descriptor: fp32 accumulator, 16-bit operands (format 0 = fp16,
// 1 = bf16), bit 16 = B is MN-major, N/8 from bit 17, M/16 from bit 24.
__host__ __device__ constexpr uint32_t idesc(int fmt, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kT >> 4) << 24);
}
// Shared-memory descriptors, 128-byte swizzle.  K-major (Q, K): 8-row groups
// 1024 bytes apart.  MN-major (V): 8-key groups 1024 bytes apart (stride
// offset), the next 64 channels a box further (leading offset).
OSSM_DEV uint64_t sdesc(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// One lane of a converged warp.
OSSM_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
OSSM_DEV void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(id), "r"(acc)
      : "memory");
}
OSSM_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(bd), "r"(id), "r"(acc)
      : "memory");
}
OSSM_DEV void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// 32 columns of this thread's lane, without the wait.
OSSM_DEV void tmem_ld32_nowait(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
// Orders uses of v after the wait before it (the load's registers are not
// valid until then, which the compiler cannot know).
OSSM_DEV void pin32(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                    "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]));
  asm volatile("" : "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                    "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]));
  asm volatile("" : "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}
// One column of this thread's lane.
OSSM_DEV uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t u;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(u)
               : "r"(taddr)
               : "memory");
  return u;
}
// 16 columns of this thread's lane times f, in place.
OSSM_DEV void tmem_scale16(uint32_t taddr, float f) {
  uint32_t u[16];
  tmem_ld16_nowait(taddr, u);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    asm volatile("" : "+r"(u[i]));
    u[i] = __float_as_uint(__uint_as_float(u[i]) * f);
  }
  tmem_st16(taddr, u);
}
OSSM_DEV void tmem_st32(uint32_t taddr, const float* v) {
  uint32_t u[16];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[16 * h + i]);
    tmem_st16(taddr + 16 * h, u);
  }
}

// The largest of three, NaN if one is.
OSSM_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// w = 2^(c x - ms) for a row's 128 scores, packed to the type; returns their
// fp32 sum.
template <typename T>
OSSM_DEV float weights(const float (&x)[kT], float c, float ms, uint32_t (&w)[kT / 2]) {
  const float2 c2 = make_float2(c, c), m2 = make_float2(-ms, -ms);
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
  for (int i = 0; i < kT / 2; ++i) {
    float2 y = fma2(make_float2(x[2 * i], x[2 * i + 1]), c2, m2);
    y = make_float2(ex2(y.x), ex2(y.y));
    if (i & 1)
      s1 = add2(s1, y);
    else
      s0 = add2(s0, y);
    w[i] = pack2<T>(y.x, y.y);
  }
  s0 = add2(s0, s1);
  return s0.x + s0.y;
}

// Does the predicate hold in any of the n threads that meet at barrier id?
OSSM_DEV bool meet_any(uint32_t id, uint32_t n, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

OSSM_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {  // has the phase passed? (may doze off for a moment)
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
constexpr long long kWaitCycles = 1LL << 31;  // about a second
// A wait that ran out ends the role; the others run out in turn.
struct Failed {
  int* flag;
  OSSM_DEV bool one(uint64_t* bar, uint32_t parity) const {  // one thread; true: give up
    if (mbar_test(bar, parity)) return false;
    const long long t0 = clock64();
    while (!mbar_test(bar, parity))
      if (clock64() - t0 > kWaitCycles) {
        *flag = 1;
        return true;
      }
    return false;
  }
  OSSM_DEV bool operator()(uint64_t* bar, uint32_t parity) const {  // a whole warp, of one mind
    if (__all_sync(~0u, mbar_test(bar, parity))) return false;
    const long long t0 = clock64();
    while (!__all_sync(~0u, mbar_test(bar, parity)))
      if (__any_sync(~0u, clock64() - t0 > kWaitCycles)) {
        *flag = 1;
        return true;
      }
    return false;
  }
};

// An arrival under a predicate, without a branch.
OSSM_DEV void mbar_arrive_if(uint64_t* bar, bool pred) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"((uint32_t)pred)
      : "memory");
}
// The waits of warps that also meet at named barriers: one that ran out is
// remembered (dead) and the warp goes on without waiting, so that the others
// are not left at a barrier; they agree to stop at the next piece.
struct Waits {
  const Failed& f;
  bool dead;
  OSSM_DEV void operator()(uint64_t* bar, uint32_t parity) {
    if (!dead) dead = f.one(bar, parity);
    __syncwarp();
  }
};

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_prompt_kernel(const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mK,
                       const __grid_constant__ CUtensorMap mV, const __grid_constant__ Params p,
                       const int lg) {  // log2 of g
  using C = Cfg<HDP>;
  constexpr int NS = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *kring = smem + 2 * C::kTile, *vring = kring + NS * C::kTile;
  __shared__ Bars bars;
  __shared__ Piece pieces[kPieces];
  __shared__ i64 pre[kGroups + 1];
  __shared__ int scalar[2];  // a tile's softmax has added its output itself
  __shared__ uint32_t tslot;
  __shared__ int failed, last_in[2];
  __shared__ unsigned long long n_items;
  __shared__ i64 cuts[2];
  __shared__ Sched::Item item;  // the first one, if item_in
  __shared__ bool item_in;

  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, cta = blockIdx.x;

  // ------------------------------------------------------------ schedule
  const int gsz = (p.B + kGroups - 1) / kGroups, ngroups = (p.B + gsz - 1) / gsz;
  const int units = p.H >> lg;
  if (threadIdx.x == 0) {
    n_items = 0;
    failed = 0;
  }
  __syncthreads();
  unsigned long long mine = 0;
  for (int g = threadIdx.x; g < ngroups; g += kThreads) {
    i64 len = 0;
    for (int b = g * gsz; b < min(p.B, (g + 1) * gsz); ++b) {
      const Shape f = shape_of(p, seq_of(p, b), lg);
      len += f.before(f.nblk) * units;
      mine += (unsigned long long)f.nblk * units;
    }
    pre[g + 1] = len;
  }
  mine = warp_sum(mine);
  if (lane == 0 && mine) atomicAdd(&n_items, mine);
  __syncthreads();
  if (warp == 0) {  // prefix sums, 32 groups at a time
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
  Sched sc{p, pre, ngroups, gsz, lg, units, {pre[ngroups], 0}};
  // CTAs for pieces of 8 key tiles; and twice the items, so that each item's
  // edge is the nearest one to some cut and short items get a CTA each
  sc.cuts.ncta = (int)min((i64)gridDim.x, max(2 * (i64)n_items, sc.cuts.total / 8));
  if (cta >= sc.cuts.ncta) return;
  if (threadIdx.x == 9 * 32) cuts[0] = sc.cut(cta, item, item_in);
  if (threadIdx.x == 10 * 32) cuts[1] = sc.cut(cta + 1);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.q_full[t], 1);
      mbar_init(&bars.q_empty[t], 1);
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.s_free[t], 4);
      mbar_init(&bars.p_ready[t], 4);
      mbar_init(&bars.pv_done[t], 1);
    }
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&bars.piece_full[i], 1);
      mbar_init(&bars.piece_empty[i], 11);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 2);
    }
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&tslot, C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  const Failed gave_up{&failed};

  // 256 x 216 + 128 x 72 = 384 x 168 registers.  With 200 and 104 the softmax
  // spilled within its loop (16384 causal, 8 heads of 64: 448 us against 388).
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {
      // ---------------------------------------------------------- schedule and loads
      if (lane == 0) {
        prefetch_tmap(&mQ);
        prefetch_tmap(&mK);
        prefetch_tmap(&mV);
        const i64 end = cuts[1];
        i64 pos = cuts[0];
        int n = 0, nq[2] = {0, 0};
        uint32_t ki = 0, vi = 0;  // K and V tiles loaded; V runs one behind
        bool ok = true;
        auto load = [&](bool v, int head, int row) {
          const uint32_t i = v ? vi++ : ki++, r = i % NS;
          uint64_t* full = v ? &bars.v_full[r] : &bars.k_full[r];
          if (i >= NS && gave_up.one(v ? &bars.v_empty[r] : &bars.k_empty[r], ((i / NS) & 1) ^ 1)) {
            --(v ? vi : ki);
            return false;
          }
          mbar_expect_tx(full, C::kTile);
          for (int x = 0; x < C::kBoxes; ++x)
            tma_load_3d((v ? vring : kring) + r * C::kTile + x * kBox, v ? &mV : &mK, full, 64 * x, head, row);
          return true;
        };
        for (;; ++n) {
          const int sl = n % kPieces;
          if (n >= kPieces && gave_up.one(&bars.piece_empty[sl], ((n / kPieces) & 1) ^ 1)) {
            ok = false;
            break;
          }
          Piece& c = pieces[sl];
          c.live = 0;
          while (pos < end) {  // the next piece with work
            const Sched::Item x = item_in ? item : sc.at(pos);
            item_in = false;
            const int a = (int)min(pos - x.start, (i64)x.n()), b = (int)min(end - x.start, (i64)x.n());
            const bool head = pos == x.start;
            pos = min(end, x.end());
            if (a >= b && !(head && x.n() == 0)) continue;
            c.live = 1;
            c.q0 = x.q.q0, c.k0 = x.q.k0, c.nk = x.q.nk, c.off = x.q.nk - x.q.nq;
            c.nrows = x.q.nq << lg;
            c.head = x.unit << lg;
            c.row0 = x.blk * 2 * kT;
            const int base = x.f.lo(x.blk);
            c.j0 = base + a, c.j1 = base + b;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
              const int row0 = c.row0 + t * kT, first = (row0 >> lg) + c.off;
              const int top = ((min(row0 + kT, c.nrows) - 1) >> lg) + c.off;
              int lo = p.window ? max(0, first - p.window + 1) >> kLT : 0, hi = top < 0 ? 0 : (top >> kLT) + 1;
              if (row0 >= c.nrows) hi = lo = 0;
              c.lo[t] = max(lo, c.j0);
              c.hi[t] = max(c.lo[t], min(hi, c.j1));
              c.w0[t] = p.window ? ((top - p.window) >> kLT) + 1 : 0;
              c.w1[t] = (first + 1) >> kLT;
            }
            c.split = b - a < x.n();
            if (c.split) {
              c.len = x.n();
              c.start = x.start;
              c.slot = head ? 2 * cta + 1 : 2 * cta;
              c.first = head ? cta : sc.cuts.first_of(x.start, x.end());
            }
            break;
          }
          mbar_arrive(&bars.piece_full[sl]);
          if (!c.live) break;
          const int kvh = c.head / (p.H / p.Hkv);
          for (int j = c.j0; j < c.j1 && ok; ++j) {
            if (j == c.j0)
#pragma unroll 1
              for (int t = 0; t < 2 && ok; ++t) {
                if (c.lo[t] >= c.hi[t]) continue;
                if (nq[t] && gave_up.one(&bars.q_empty[t], (nq[t] & 1) ^ 1)) {
                  ok = false;
                  break;
                }
                ++nq[t];
                mbar_expect_tx(&bars.q_full[t], C::kTile);
                for (int x = 0; x < C::kBoxes; ++x)
                  tma_load_3d(smem + t * C::kTile + x * kBox, &mQ, &bars.q_full[t], 64 * x, c.head,
                              c.q0 + ((c.row0 + t * kT) >> lg));
              }
            ok = ok && load(false, kvh, c.k0 + j * kT) && (j == c.j0 || load(true, kvh, c.k0 + (j - 1) * kT));
          }
          if (c.j0 < c.j1) ok = ok && load(true, kvh, c.k0 + (c.j1 - 1) * kT);
          if (!ok) break;
        }
        if (!ok) {  // no copy may still be landing when the CTA exits
          for (int t = 0; t < 2; ++t)
            if (nq[t]) gave_up.one(&bars.q_full[t], (nq[t] & 1) ^ 1);
          for (uint32_t i = ki > NS ? ki - NS : 0; i < ki; ++i) gave_up.one(&bars.k_full[i % NS], (i / NS) & 1);
          for (uint32_t i = vi > NS ? vi - NS : 0; i < vi; ++i) gave_up.one(&bars.v_full[i % NS], (i / NS) & 1);
        }
      }
    } else if (warp == 8) {
      // ---------------------------------------------------------- S_t = Q_t K^T
      // Scores and outputs are issued by a warp each: one for both was busy with
      // its waits and left the tensor core idle.  The whole warp walks the loop,
      // so that operands stay uniform; one lane issues.
      constexpr uint32_t id = idesc(std::is_same<T, __half>::value ? 0 : 1, kT, 0);
      const bool leader = elect_one();
      const uint32_t qb = smem_u32(smem), kb = smem_u32(kring);
      uint32_t nq[2] = {0, 0}, ns[2] = {0, 0}, g = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int sl = n % kPieces;
        if (gave_up(&bars.piece_full[sl], (n / kPieces) & 1)) break;
        const Piece& c = pieces[sl];
        if (!c.live) break;
        const int j1 = c.j1, lo[2] = {c.lo[0], c.lo[1]}, hi[2] = {c.hi[0], c.hi[1]};
        int j = c.j0;
        __syncwarp();
        if (leader) mbar_arrive(&bars.piece_empty[sl]);
        for (; j < j1 && ok; ++j, ++g) {
          const uint32_t r = g % NS;
          if (gave_up(&bars.k_full[r], (g / NS) & 1)) {
            ok = false;
            break;
          }
          const uint64_t kd = sdesc(kb + r * C::kTile, 16);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j < lo[t] || j >= hi[t]) continue;
            constexpr int kS = C::kS;
            const int b = t % kS;
            if ((j == lo[t] && gave_up(&bars.q_full[t], nq[t]++ & 1)) ||
                (ns[b] && gave_up(&bars.s_free[b], (ns[b] & 1) ^ 1))) {
              ok = false;
              break;
            }
            ++ns[b];
            tc_fence_after();
            if (leader) {
              const uint64_t qd = sdesc(qb + t * C::kTile, 16);
#pragma unroll
              for (int kk = 0; kk < HDP / 16; ++kk) {
                const uint32_t o = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
                mma_ss(tmem + b * kT, qd + o, kd + o, id, kk > 0);
              }
              mma_commit(&bars.s_full[t]);
              if (j == hi[t] - 1) mma_commit(&bars.q_empty[t]);
            }
          }
          if (leader) mma_commit(&bars.k_empty[r]);
        }
      }
      if (!ok) failed = 1;
    } else {
      // ---------------------------------------------------------- O_t += P_t V
      constexpr uint32_t id = idesc(std::is_same<T, __half>::value ? 0 : 1, HDP, 1);
      const bool leader = elect_one();
      const uint32_t vb = smem_u32(vring);
      const int t = warp - 10;
      uint32_t np = 0, g = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int sl = n % kPieces;
        if (gave_up(&bars.piece_full[sl], (n / kPieces) & 1)) break;
        const Piece& c = pieces[sl];
        if (!c.live) break;
        const int j1 = c.j1, lo = c.lo[t], hi = c.hi[t];
        int j = c.j0;
        __syncwarp();
        if (leader) mbar_arrive(&bars.piece_empty[sl]);
        for (; j < j1; ++j, ++g) {
          const uint32_t r = g % NS;
          const bool act = j >= lo && j < hi;
          if (gave_up(&bars.v_full[r], (g / NS) & 1) || (act && gave_up(&bars.p_ready[t], np++ & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (leader) {
            if (act) {
              if (!*(volatile int*)&scalar[t]) {
                const uint64_t vd = sdesc(vb + r * C::kTile, kBox);
#pragma unroll
                for (int kk = 0; kk < kT / 16; ++kk)
                  mma_ts(tmem + C::kO + t * HDP, tmem + C::kP + t * (kT / 2) + kk * 8, vd + kk * (2048 >> 4), id,
                         kk > 0 || j > lo);
              }
              mma_commit(&bars.pv_done[t]);
            }
            mma_commit(&bars.v_empty[r]);
          }
          __syncwarp();
        }
      }
      if (!ok) failed = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------------------------------------------------- softmax and output
    const int t = warp >> 2, row = threadIdx.x & (kT - 1);
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), tS = tl + (t % C::kS) * kT,
                   tP = tl + C::kP + t * (kT / 2), tO = tl + C::kO + t * HDP;
    uint32_t ns = 0, npv = 0, it = 0;  // score tiles seen, outputs waited for, steps before the piece
    Waits wait{gave_up, false};
    auto settled = [&](uint32_t upto) {  // the outputs of all score tiles before this one are in
      if (npv == upto) return;
      wait(&bars.pv_done[t], npv & 1);
      ++npv;
      tc_fence_after();
    };
    auto free_scores = [&]() {
      tc_fence_before();
      __syncwarp();
      mbar_arrive_if(&bars.s_free[t % C::kS], lane == 0);
    };
    for (int n = 0;; ++n) {
      const int sl = n % kPieces;
      wait(&bars.piece_full[sl], (n / kPieces) & 1);
      if (meet_any(1 + t, kT, wait.dead)) break;
      const Piece& c = pieces[sl];  // given back at the piece's end
      if (!c.live) break;
      const int lo = c.lo[t], hi = c.hi[t], j0 = c.j0;
      const int row0 = c.row0 + t * kT;
      int w0 = c.w0[t], w1 = c.w1[t], at = ((row0 + row) >> lg) + c.off;  // the row's position
      asm volatile("" : "+r"(w0), "+r"(w1), "+r"(at));  // in registers, not worked out again for every tile
      float m = -INFINITY, l = 0.f;
      for (int j = lo; j < hi; ++j) {
        wait(&bars.s_full[t], ns & 1);
        ++ns;
        tc_fence_after();
        float x[kT];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(tS + 32 * i, x + 32 * i);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) pin32(x + 32 * i);
        free_scores();
        const bool part = j < w0 || j >= w1;
        const int k_hi = at - j * kT, k_lo = p.window ? k_hi - p.window + 1 : -1;  // seen: k_lo <= key <= k_hi
        if (part) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // bit e: key 32 i + e is seen
            const int a = k_lo - 32 * i, b = k_hi - 32 * i;
            const uint32_t up = b >= 31 ? ~0u : b < 0 ? 0u : (2u << b) - 1u;
            const uint32_t seen = up & (a <= 0 ? ~0u : a > 31 ? 0u : ~0u << a);
#pragma unroll
            for (int e = 0; e < 32; ++e) x[32 * i + e] = (seen >> e & 1u) ? x[32 * i + e] : -INFINITY;
          }
        }
        float mx[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = max3(x[16 * i], x[16 * i + 1], x[16 * i + 2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2)
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i] = max3(mx[i], x[16 * i + e], x[16 * i + e + 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx[i] = max3(max3(mx[i], mx[i + 4], x[16 * i + 15]), x[16 * i + 79], x[16 * i + 79]);
        mx[0] = max3(mx[0], mx[1], mx[2]);
        const float top = max3(mx[0], mx[3], mx[3]) * p.scale2;
        if (!(top < INFINITY)) m = NAN;  // a seen score is NaN or infinite: so is the softmax's sum
        const bool grow = top > m + 8.f;
        if (__any_sync(~0u, grow)) {
          const float mn = grow ? top : m;
          const float f = grow ? ex2(m - mn) : 1.f;
          m = mn;
          l *= f;
          if (j > lo) {
            settled(ns - 1);
#pragma unroll 1
            for (int i = 0; i < HDP / 16; ++i) tmem_scale16(tO + 16 * i, f);
          }
        }
        const float ms = m == -INFINITY ? 0.f : m;  // a row that has seen no key yet
        uint32_t w[kT / 2];
        l += weights<T>(x, p.scale2, ms, w);
        settled(ns - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) u[e] = w[16 * i + e];
          tmem_st16(tP + 16 * i, u);
        }
        if (part) {
          const uint32_t g = it + (j - j0);
          wait(&bars.v_full[g % NS], (g / NS) & 1);
          // A weight of 0 times NaN is NaN: V rows past the sequence become
          // zeros, and if another one holds a non-finite value, the product
          // is taken here over the seen keys alone.
          uint4* vr = reinterpret_cast<uint4*>(vring + (g % NS) * C::kTile + row * 128);
          uint32_t big = 0;  // the largest magnitudes, as packed integers: NaN and infinities are above all others
          if (j * kT + row < c.nk) {
#pragma unroll
            for (int i = 0; i < 8 * C::kBoxes; ++i) {  // in an order that spreads the rows over the banks
              const uint4 u = vr[(i >> 3) * (kBox / 16) + ((i ^ row) & 7)];
              big = __vmaxu2(__vmaxu2(big, u.x & 0x7fff7fffu), u.y & 0x7fff7fffu);
              big = __vmaxu2(__vmaxu2(big, u.z & 0x7fff7fffu), u.w & 0x7fff7fffu);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8 * C::kBoxes; ++i)
              vr[(i >> 3) * (kBox / 16) + ((i ^ row) & 7)] = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();  // before the tensor core reads them
          }
          const bool own = meet_any(1 + t, kT, nonfinite2<T>(big));
          if (row == 0) scalar[t] = own;
          if (own) {
            tmem_wait_st();
            const uint8_t* vt = vring + (g % NS) * C::kTile;
#pragma unroll 1
            for (int i = 0; i < HDP / 32; ++i) {
              float o[32];
              if (j > lo) {
                tmem_ld32_nowait(tO + 32 * i, o);
                tmem_wait_ld();
                pin32(o);
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
              }
              const uint8_t* vb = vt + (i >> 1) * kBox;
#pragma unroll 1
              for (int k = 0; k < kT; ++k) {
                const float2 w2 = to_f2<T>(tmem_ld1(tP + (k >> 1)));
                const float w = (k & 1) ? w2.y : w2.x;
                if (k >= k_lo && k <= k_hi) {
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    const float2 v2 = to_f2<T>(*reinterpret_cast<const uint32_t*>(
                        vb + k * 128 + ((((i & 1) * 64 + e * 4)) ^ ((k & 7) << 4))));
                    o[2 * e] = fmaf(w, v2.x, o[2 * e]);
                    o[2 * e + 1] = fmaf(w, v2.y, o[2 * e + 1]);
                  }
                }
                __syncwarp();
              }
              tmem_st32(tO + 32 * i, o);
            }
          }
        }
        if (!part && row == 0) scalar[t] = 0;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&bars.p_ready[t], lane == 0);
      }
      it += c.j1 - j0;
      settled(ns);
      const bool mine_row = row0 + row < c.nrows;
      T* out = static_cast<T*>(p.out) + (i64)(c.q0 + ((row0 + row) >> lg)) * p.ost +
               (i64)(c.head + ((row0 + row) & ((1 << lg) - 1))) * p.osh;
      if (!c.split) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int i = 0; i < HDP / 32; ++i) {
          float o[32];
          if (hi > lo) {
            tmem_ld32_nowait(tO + 32 * i, o);
            tmem_wait_ld();
            pin32(o);
          }
          if (mine_row) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (32 * i + 8 * e >= p.hd) break;
              uint4 u = make_uint4(0, 0, 0, 0);
              if (hi > lo && l != 0.f) {
                u.x = pack2<T>(o[8 * e] * inv, o[8 * e + 1] * inv);
                u.y = pack2<T>(o[8 * e + 2] * inv, o[8 * e + 3] * inv);
                u.z = pack2<T>(o[8 * e + 4] * inv, o[8 * e + 5] * inv);
                u.w = pack2<T>(o[8 * e + 6] * inv, o[8 * e + 7] * inv);
              }
              *reinterpret_cast<uint4*>(out + 32 * i + 8 * e) = u;
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        if (lane == 0) mbar_arrive(&bars.piece_empty[sl]);
        continue;
      }
      // a piece of an item: (m, l, O) to the workspace; float4 e of every row side by side
      float* mine_part = p.part + (size_t)c.slot * C::kPartFloats;
      const int r2 = t * kT + row;
      const bool any = hi > lo;
      if (mine_row) {
        mine_part[r2] = m;
        mine_part[2 * kT + r2] = l;
      }
      float4* po = reinterpret_cast<float4*>(mine_part + 4 * kT);
#pragma unroll 1
      for (int i = 0; i < HDP / 32; ++i) {
        float o[32];
        if (any) {
          tmem_ld32_nowait(tO + 32 * i, o);
          tmem_wait_ld();
          pin32(o);
        }
        if (mine_row) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            po[(8 * i + e) * 2 * kT + r2] =
                any ? make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncwarp();
      }
      tc_fence_before();
      __threadfence();
      // the tiles join apart: neither softmax may wait for the other here, whose
      // products can be queued behind this one's next scores
      named_sync(1 + t, kT);
      if (row == 0) {
        uint32_t* count = p.counts + 2 * c.first + t;
        const uint32_t done = atomicAdd(count, (uint32_t)(c.j1 - c.j0)) + (c.j1 - c.j0);
        last_in[t] = done == (uint32_t)c.len;
        if (last_in[t]) *count = 0;  // for the next call
      }
      named_sync(1 + t, kT);
      if (!last_in[t]) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.piece_empty[sl]);
        continue;
      }
      __threadfence();
      // The last one in joins the pieces in the order of the cut: a thread takes
      // 8 channels of a row at a time, 8 pieces' worth of loads ahead.
      const int np = sc.cuts.last_of(c.start, c.start + c.len + kItemCost, c.start + c.len - 1) - c.first + 1;
      const int rows = min(kT, c.nrows - row0);
      for (int e = row; e < rows * (p.hd / 8); e += kT) {
        const int r = e % rows, d = e / rows * 8, rr = t * kT + r;
        float M = -INFINITY, L = 0.f, acc[8] = {};
        for (int k0 = 0; k0 < np; k0 += 8) {
          float pm[8], pl[8];
          float4 u[8], v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            pm[k] = -INFINITY, pl[k] = 0.f;
            u[k] = v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + k < np) {
              const float* q = p.part + (size_t)(k0 + k ? 2 * (c.first + k0 + k) : 2 * c.first + 1) * C::kPartFloats;
              const float4* qo = reinterpret_cast<const float4*>(q + 4 * kT) + (d / 4) * 2 * kT + rr;
              pm[k] = __ldcg(q + rr);
              pl[k] = __ldcg(q + 2 * kT + rr);
              u[k] = __ldcg(qo);
              v[k] = __ldcg(qo + 2 * kT);
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
        const float inv = L == 0.f ? 0.f : 1.f / L;
        T* to = static_cast<T*>(p.out) + (i64)(c.q0 + ((row0 + r) >> lg)) * p.ost +
                (i64)(c.head + ((row0 + r) & ((1 << lg) - 1))) * p.osh;
        *reinterpret_cast<uint4*>(to + d) =
            make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                       pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.piece_empty[sl]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
  if (threadIdx.x == 0 && failed) atomicExch(&p.hdr->status, (uint32_t)OSSM_ETIMEOUT);
}

// [rows, heads, hd] as (channel, head, row); box: 64 channels of g heads of
// 128 / g rows; channels past hd and rows past the end read as zero.
bool encode(CUtensorMap* map, int dtype, const void* base, int hd, int heads, i64 rows, i64 st, i64 sh, int g) {
  // a single row or head has no stride of its own to respect
  if (heads == 1) sh = hd;
  if (rows == 1) st = std::max(st, (i64)heads * std::max(sh, (i64)hd));
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)g, (cuuint32_t)(kT / g)};
  cuuint32_t estr[3] = {1, 1, 1};
  return fast::encode_fn()(map, dtype == OSSM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HDP>
cudaError_t launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p, int lg, int grid,
                   cudaStream_t st) {
  auto kern = attn_prompt_kernel<T, HDP>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kern, (int)Cfg<HDP>::kSmem, done);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, Cfg<HDP>::kSmem, st>>>(q, k, v, p, lg);
  return cudaGetLastError();
}

size_t prompt_part_floats(int hd) { return 2 * (hd <= 64 ? Cfg<64>::kPartFloats : Cfg<128>::kPartFloats); }

int prompt_forward(const ossm_attn_args* a, const Params& p, int grid, cudaStream_t st) {
  if (!fast::encode_fn()) return OSSM_ELAUNCH;
  CUtensorMap q, k, v;
  // Two heads a tile where there are two, more only as far as the queries do
  // not fill the item's rows: 3 x 4096 causal, 32/8 heads of 128, was 3 % faster
  // with 2 than with 4; 32 x 5 new tokens against 8192 took 229 us with 4 and
  // 487 us with one a tile.
  int lg = 0;
  while (lg < 7 && (p.H / p.Hkv) % (2 << lg) == 0 && (lg == 0 || ((int64_t)a->max_seqlen_q << lg) < 2 * kT)) ++lg;
  if (!encode(&q, a->dtype, p.q, p.hd, p.H, p.Tq, p.qst, p.qsh, 1 << lg) ||
      !encode(&k, a->dtype, p.k, p.hd, p.Hkv, p.Tk, p.kst, p.ksh, 1) ||
      !encode(&v, a->dtype, p.v, p.hd, p.Hkv, p.Tk, p.vst, p.vsh, 1))
    return OSSM_EINVAL;
  const bool bf = a->dtype == OSSM_BF16;
  cudaError_t e;
  if (p.hd <= 64)
    e = bf ? launch<__nv_bfloat16, 64>(q, k, v, p, lg, grid, st) : launch<__half, 64>(q, k, v, p, lg, grid, st);
  else
    e = bf ? launch<__nv_bfloat16, 128>(q, k, v, p, lg, grid, st) : launch<__half, 128>(q, k, v, p, lg, grid, st);
  return e == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

}  // namespace attn
}  // namespace ossm
