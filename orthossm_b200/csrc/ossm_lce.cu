// The language-model loss from hidden states: softmax cross entropy over the
// vocabulary of the logits z = H W^T, and its gradients, without keeping z.
//
//   lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_t,target + zl lse_t^2
//   dz_tv = g_t ((1 + 2 zl lse_t) exp(z_tv - lse_t) - [v = target]),
//   dH = dZ W,  dW = dZ^T H
//
// Forward: rows (which tokens have a target, their states side by side), stats
// (logits tile by tile on the tensor core, a running maximum and sum a row),
// finish (joins the sums, the losses and their sum).  Backward: rows, then for
// each piece of the vocabulary gradz (the logits again, dz rounded to the
// inputs' type into the workspace), prod (dW of the piece, dH) and join (the
// tiles that several CTAs made parts of).
//
// Tokens without a target have no part in any product: their states are not
// read, so NaN there harms nothing, and they cost nothing.
//
// dz is rounded to the inputs' 16 bits, as the tensor core takes it: gradients are
// 1.1 to 1.5 times as far from float64 as fp32 products leave them (up to 2.7 and
// 7.6 times, dH and dW, for single tokens, where its largest entry is everything).
// The logits' sums are the tensor core's, which cut where fp32 rounds: a loss is off
// by 2e-7 of its value at 512 channels, 6e-7 (one token: 1e-5) at 2000.
//
// What bounds it: the tensor pipe, 8 T d V operations where keeping the logits
// would take 6, and in long runs the power cap.  Measured in bursts, 16384
// tokens, 512 channels, 32000 columns, bf16: stats 316 to 324 us (1625 to 1665
// TFLOP/s, the pipe 97 % busy), gradz 439 to 454 (its dz, a gigabyte, costs 100 of
// them), the products 786 to 821 and their joins 42 to 44; 8192, 2048, 131072: 2872 to 2910, 3076 to 3160, 6843 to
// 6949 and 87 to 92 us (1511 to 1531, 1392 to 1430, 1266 to 1286 TFLOP/s).
// Tried: pieces of 32 to 256 MB (3 to 60 % slower), A's tile resident (2 % in a
// timing probe at 512 channels), one CTA a tile (6 to 17 % slower in the products).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "ossm_attn.cuh"
#include "ossm_sm100.cuh"

namespace ossm {
int device_sms();
namespace fast {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
}
namespace lce {

using namespace sm100;
using attn::allow_smem;
using attn::ex2;
using attn::pack2;
typedef long long i64;

// A tile of 256 x 256 is made by the two CTAs of a cluster (cta_group::2): each
// loads 128 rows of A and 128 of B and holds 128 rows of sums, and one issues the
// products for both.  A stage is 32 KB and feeds 512 cycles of the tensor core;
// with a CTA alone on 128 x 256 it was 48 KB, and four stages did not cover the
// way from HBM (tensor pipe 61 % busy in the products with dz, 1.57 GHz).
constexpr int kM = 256, kN = 256, kK = 64;  // a tile, and the depth of one load
constexpr int kHalf = 128;                  // rows of A and of B that a CTA loads
constexpr int kThreads = 320;               // 8 warps read tensor memory, one loads, one issues products
constexpr int kABytes = kHalf * kK * 2, kStage = 2 * kABytes;
constexpr int kOutZ = 8 * 2 * 32 * 128;     // gradz: two [32 rows x 64 columns] boxes a warp
constexpr int kOutP = 8 * 32 * 64;          // the products: a [32 rows x 32 columns] box a warp
constexpr int kStages = 6, kStagesZ = 5;
constexpr size_t smem_bytes(int stages, int out) { return stages * (size_t)kStage + out + 1024; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowThreads = 1024;
constexpr int kMaxBlocks = 1024;

struct Head {      // of the workspace
  int n;           // tokens that have a target
  float unit;      // backward: what dz in the workspace is in units of
  uint32_t count;  // finished blocks
};
// dz is written in units that bring the largest factor of all rows to kDzScale:
// its row's probabilities down to 2^-28 stay out of fp16's subnormals, whatever the
// loss was multiplied by, and those down to 2^-28 / rho of a row with a share rho
// of that factor.  One unit, as dW sums over rows.  (bf16 has the exponents, but
// one rule does.)
constexpr float kDzScale = 16384.f;

struct Params {
  i64 T;
  int Tpad, d, V;
  const void* hidden;
  i64 hst;
  const int64_t* targets;
  i64 ignore;
  float zl;
  int reduction;
  float *loss, *lse, *rest;
  const float* g;
  void *dh, *dw;
  Head* head;
  int *rows, *tgt;   // [n] token and target of each row
  float *lse2, *fa, *fb;  // [n] lse log2(e), factors of the softmax and of the target
  void* hc;          // [Tpad, dst] states of the rows side by side, where tokens were left out
  int dst;           // d up to whole 128 bytes: the copies are read by lines
  float2* part;      // [Tpad, 2 * panels] maximum (base 2) and sum of a row over a panel's half columns
  float* zt;         // [Tpad] the target's logit
  double* sums;      // [kMaxBlocks]
  float* dh32;       // [tiles] sums of dH over the pieces, in the order of tensor memory
  float* cuts;       // [2 a CTA] sums of tiles that are cut, the same
  int panels, pan;   // panels of `pan` tiles of columns
  int v0, vp;        // the piece: columns v0 .. v0 + vp
  int first, last;   // the piece is the first, the last
  uint32_t* status;
};

// ---------------------------------------------------------------- waits
OSSM_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
constexpr i64 kWaitCycles = 1LL << 31;  // about a second
// True: it ran out.  The role then goes on without waiting (readers of tensor
// memory) or ends; the others run out in turn.
OSSM_DEV bool gave_up(uint64_t* bar, uint32_t parity, int* failed) {
  if (mbar_test(bar, parity)) return false;
  const i64 t0 = clock64();
  while (!mbar_test(bar, parity))
    if (clock64() - t0 > kWaitCycles) {
      *failed = 1;
      return true;
    }
  return false;
}

OSSM_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
OSSM_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of a barrier of the pair's first CTA.
OSSM_DEV uint32_t first_cta(const uint64_t* bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
  return r;
}
// Orders nothing in memory: what is handed over is tensor memory that has been
// read (a release at cluster scope stalled the readers' warps).
OSSM_DEV void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Into this CTA's shared memory, counted by a barrier of the pair's first CTA.
OSSM_DEV void tma_load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
OSSM_DEV void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
OSSM_DEV void bulk_wait0() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Instruction descriptor: fp32 accumulator, 16-bit operands (0 = fp16, 1 =
// bf16), bits 15 and 16: A, B are MN-major, N/8 from bit 17, M/16 from bit 24.
__host__ __device__ constexpr uint32_t idesc(int fmt, int a_mn, int b_mn, int n) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
// Shared-memory descriptor, 128-byte swizzle.  K-major: groups of 8 rows 1024
// bytes apart.  MN-major: groups of 8 steps of K 1024 bytes apart, the next 64
// of M or N a box of 64 x 64 further.
constexpr int kBox = 64 * 128;
OSSM_DEV uint64_t sdesc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)(kBox >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
OSSM_DEV void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(id), "r"(acc)
      : "memory");
}
// Arrives at the barrier of this place in both CTAs once the products are done.
OSSM_DEV void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
OSSM_DEV void pair_alloc(uint32_t* slot) {  // whole warp, in both CTAs: all columns
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
OSSM_DEV void pair_dealloc(uint32_t taddr) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}
OSSM_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
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
// Orders uses of v after the wait before it.
OSSM_DEV void pin32(float* v) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}

// ---------------------------------------------------------------- what the tensor-core kernels share
template <int S>
struct Shared {
  uint64_t full[S], empty[S], acc_full[2], acc_empty[2];  // full, acc_empty: those of the first CTA are used
  uint32_t tmem;
  int failed;
};

// Barriers, tensor memory: all threads, before the roles part.
template <int S>
OSSM_DEV void setup(Shared<S>& s, int warp) {
  if (threadIdx.x == 0) {
    s.failed = 0;
    for (int i = 0; i < S; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 16);
    }
    fence_mbar_init();
  }
  if (warp == 9) pair_alloc(&s.tmem);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
}
template <int S>
OSSM_DEV void teardown(Shared<S>& s, int warp, uint32_t* status) {
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA's memory goes before the other is through
  if (warp == 9) {
    tc_fence_after();
    pair_dealloc(s.tmem);
  }
  if (threadIdx.x == 0 && s.failed && status) atomicExch(status, (uint32_t)OSSM_ETIMEOUT);
}

// The ring of loaded stages, on the loading side of either CTA.
template <int S>
struct Loader {
  Shared<S>& s;
  uint8_t* ring;
  bool first;  // the pair's first CTA expects the bytes of both
  uint32_t r, turn, n;
  OSSM_DEV uint8_t* next(uint32_t bytes, uint32_t& bar) {  // NULL: give up
    if (n >= S && gave_up(&s.empty[r], turn ^ 1, &s.failed)) return nullptr;
    if (first) mbar_expect_tx(&s.full[r], 2 * bytes);
    bar = first_cta(&s.full[r]);
    uint8_t* to = ring + r * kStage;
    ++n;
    if (++r == S) r = 0, turn ^= 1;
    return to;
  }
  // No copy, and no arrival at this CTA's barriers, may be on its way when the CTAs exit.
  OSSM_DEV void end(bool ok) {
    for (uint32_t j = n > S ? n - S : 0; j < n; ++j)
      if (ok) gave_up(&s.empty[j % S], (j / S) & 1, &s.failed);
      else if (first) gave_up(&s.full[j % S], (j / S) & 1, &s.failed);
  }
};

// One tile's products: `steps` stages into the sums of this turn (the first CTA
// issues them, a whole warp walks).  a_step, b_step: bytes between the starts of
// two 16-deep products.
template <int S>
struct Issuer {
  Shared<S>& s;
  uint32_t ring, r, turn, tiles;
  OSSM_DEV bool tile(int steps, uint32_t id, uint32_t a_step, uint32_t b_step, bool leader) {
    const uint32_t b = tiles & 1;
    if (tiles >= 2 && __any_sync(~0u, gave_up(&s.acc_empty[b], ((tiles >> 1) & 1) ^ 1, &s.failed))) return false;
    tc_fence_after();
    for (int k = 0; k < steps; ++k) {
      if (__any_sync(~0u, gave_up(&s.full[r], turn, &s.failed))) return false;
      tc_fence_after();
      if (leader) {
        const uint64_t ad = sdesc(ring + r * kStage), bd = sdesc(ring + r * kStage + kABytes);
#pragma unroll
        for (int kk = 0; kk < kK / 16; ++kk)
          mma(s.tmem + b * kN, ad + kk * (a_step >> 4), bd + kk * (b_step >> 4), id, k > 0 || kk > 0);
        mma_commit(&s.empty[r]);
      }
      __syncwarp();
      if (++r == S) r = 0, turn ^= 1;
    }
    if (leader) mma_commit(&s.acc_full[b]);
    __syncwarp();
    ++tiles;
    return true;
  }
};

// ---------------------------------------------------------------- logits
enum { STATS, GRADZ };

// Items of the logits kernels: a block of 256 rows by a panel of columns.  The
// blocks stand in groups whose rows L2 keeps (32 MB); of a group all take a panel
// before the next one, so that W is read once a group.
struct Walk {
  int blocks, panels, items, group;
  OSSM_DEV Walk(const Params& p) {
    blocks = max(1, (p.head->n + kM - 1) / kM);
    panels = p.panels;
    items = blocks * panels;
    const int most = max(8, (32 << 20) / (kM * 2 * p.d)), groups = (blocks + most - 1) / most;
    group = (blocks + groups - 1) / groups;
  }
  OSSM_DEV void at(int it, int& block, int& panel) const {
    const int g = it / (group * panels), r = it - g * group * panels, rows = min(group, blocks - group * g);
    panel = r / rows;
    block = group * g + r % rows;
  }
};

template <typename T, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    lce_logits_kernel(const __grid_constant__ CUtensorMap mH, const __grid_constant__ CUtensorMap mHc,
                      const __grid_constant__ CUtensorMap mW, const __grid_constant__ CUtensorMap mZ,
                      const __grid_constant__ Params p) {
  constexpr int S = MODE == GRADZ ? kStagesZ : kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Shared<S> s;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  setup(s, warp);
  const int n = p.head->n;
  const Walk walk(p);
  const int ktiles = (p.d + kK - 1) / kK;
  const int ntiles = (min(p.vp, p.V - p.v0) + kN - 1) / kN;  // of the piece

  if (warp == 8) {
    if (lane == 0) {
      const CUtensorMap* a = n == p.T ? &mH : &mHc;
      Loader<S> ld{s, smem, rank == 0, 0, 0, 0};
      bool ok = true;
      for (int it = pair; it < walk.items && ok; it += pairs) {
        int block, panel;
        walk.at(it, block, panel);
        for (int nt = panel * p.pan; nt < min(ntiles, (panel + 1) * p.pan) && ok; ++nt)
          for (int k = 0; k < ktiles; ++k) {
            uint32_t bar;
            uint8_t* to = ld.next(kStage, bar);
            if (!to) {
              ok = false;
              break;
            }
            tma_load_2d(to, a, bar, k * kK, block * kM + rank * kHalf);
            tma_load_2d(to + kABytes, &mW, bar, k * kK, p.v0 + nt * kN + rank * kHalf);
          }
      }
      ld.end(ok);
    }
  } else if (warp == 9) {
    if (rank == 0) {
      const bool leader = elect_one();
      Issuer<S> mm{s, smem_u32(smem), 0, 0, 0};
      constexpr uint32_t id = idesc(std::is_same<T, __half>::value ? 0 : 1, 0, 0, kN);
      bool ok = true;
      for (int it = pair; it < walk.items && ok; it += pairs) {
        int block, panel;
        walk.at(it, block, panel);
        for (int nt = panel * p.pan; nt < min(ntiles, (panel + 1) * p.pan) && ok; ++nt)
          ok = mm.tile(ktiles, id, 32, 32, leader);
      }
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tl = s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 128;
    uint8_t* box = smem + S * kStage + warp * 8192;
    const uint32_t freed[2] = {first_cta(&s.acc_empty[0]), first_cta(&s.acc_empty[1])};
    uint32_t tiles = 0;
    bool dead = false;
    for (int it = pair; it < walk.items; it += pairs) {
      int block, panel;
      walk.at(it, block, panel);
      const int r = block * kM + rank * kHalf + row;
      const bool live = r < n;
      const int tcol = live ? __ldg(p.tgt + r) - p.v0 : -1;
      float ms = -INFINITY, l = 0.f;              // STATS
      float lse2 = 0.f, fa = 0.f, fb = 0.f;       // GRADZ
      if (MODE == GRADZ && live) lse2 = __ldg(p.lse2 + r), fa = __ldg(p.fa + r), fb = __ldg(p.fb + r);
      for (int nt = panel * p.pan; nt < min(ntiles, (panel + 1) * p.pan); ++nt, ++tiles) {
        const uint32_t b = tiles & 1;
        if (!dead) dead = gave_up(&s.acc_full[b], (tiles >> 1) & 1, &s.failed);
        __syncwarp();
        tc_fence_after();
        float x[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(tl + b * kN + 32 * i, x + 32 * i);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) pin32(x + 32 * i);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(freed[b]);
        const int c0 = nt * kN + half * 128;
        const int cols = min(p.V - p.v0, p.vp) - c0;  // that exist
        const int at = tcol - c0;                     // the target's place
        const bool here = __any_sync(~0u, at >= 0 && at < 128);
        if (MODE == STATS) {
          if (cols < 128) {
#pragma unroll
            for (int i = 0; i < 128; ++i) x[i] = i < cols ? x[i] : -INFINITY;
          }
          if (here) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < 128; ++i) z = i == at ? x[i] : z;
            if (at >= 0 && at < 128) p.zt[r] = z;
          }
          float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int i = 4; i < 128; i += 4) {
            mx[0] = fmaxf(mx[0], x[i]), mx[1] = fmaxf(mx[1], x[i + 1]);
            mx[2] = fmaxf(mx[2], x[i + 2]), mx[3] = fmaxf(mx[3], x[i + 3]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kLog2e;
          if (top > ms + 8.f) {  // the reference follows the maximum in steps, so that few tiles rescale
            l *= ex2(ms - top);
            ms = top;
          }
          const float off = ms == -INFINITY ? 0.f : ms;
          const float2 c2 = make_float2(kLog2e, kLog2e), m2 = make_float2(-off, -off);
          float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            float2 y = fma2(make_float2(x[2 * i], x[2 * i + 1]), c2, m2);
            y = make_float2(ex2(y.x), ex2(y.y));
            if (i & 1) s1 = attn::add2(s1, y); else s0 = attn::add2(s0, y);
          }
          s0 = attn::add2(s0, s1);
          l += s0.x + s0.y;
        } else {
          const float2 c2 = make_float2(kLog2e, kLog2e), m2 = make_float2(-lse2, -lse2);
          const float2 a2 = make_float2(fa, fa);
          if (lane == 0) bulk_wait_read0();  // the last tile's boxes have left
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 4; ++h) {
#pragma unroll
            for (int i = 16 * h; i < 16 * h + 16; ++i) {
              float2 y = fma2(make_float2(x[2 * i], x[2 * i + 1]), c2, m2);
              y = mul2(make_float2(ex2(y.x), ex2(y.y)), a2);
              x[2 * i] = y.x, x[2 * i + 1] = y.y;
            }
            if (here) {
#pragma unroll
              for (int i = 32 * h; i < 32 * h + 32; ++i) x[i] = i == at ? x[i] - fb : x[i];
            }
            if (cols < 128 || !live) {
#pragma unroll
              for (int i = 32 * h; i < 32 * h + 32; ++i) x[i] = live && i < cols ? x[i] : 0.f;
            }
#pragma unroll
            for (int i = 4 * h; i < 4 * h + 4; ++i) {
              const float* y = x + 8 * i;
              *reinterpret_cast<uint4*>(box + (i >> 3) * 4096 + lane * 128 + (((i ^ lane) & 7) << 4)) =
                  make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int to = block * kM + rank * kHalf + (warp & 3) * 32;
            tma_store_2d(&mZ, box, c0, to);
            tma_store_2d(&mZ, box + 4096, c0 + 64, to);
            bulk_commit();
          }
        }
      }
      if (MODE == STATS && live) p.part[(i64)r * 2 * p.panels + 2 * panel + half] = make_float2(ms, l);
    }
    if (MODE == GRADZ && lane == 0) bulk_wait0();
  }
  teardown(s, warp, p.status);
}

// ---------------------------------------------------------------- dW = dZ^T H of the piece, dH += dZ W
// The tiles of both products.  Whole rounds of them, one a pair of CTAs, run side
// by side, so that the pairs at work share what they read of dZ; the tiles that
// are left over stand on a line, which is cut evenly over the pairs.  A tile that
// is cut leaves sums in the workspace, which a kernel after this one adds up in
// order.  (The pair that finished last did that first: with 64 tokens and 50000
// columns, where two tiles of dH are cut into 37, it took 290 of 323 us.)  (T = 16384, 512 channels, pieces of 16384 columns: 254 tiles
// on 74 pairs, 3.43 rounds.)
constexpr int kEnd = 10;  // a tile's end (its sums read, converted, stored) takes as long as so many steps of the next
struct Tiles {
  int nt, tw, th, kw, kh;  // tiles a row of tiles, of dW, of dH; their steps
  int ncta, rw, rh, lw, lh;  // pairs; rounds, and what is left
  i64 line;
  OSSM_DEV Tiles(const Params& p, int n, int cols, int grid) {
    const int nn = max(n, 1);
    nt = (p.d + kN - 1) / kN;
    tw = p.dw ? (cols + kM - 1) / kM * nt : 0;
    th = p.dh ? (nn + kM - 1) / kM * nt : 0;
    kw = (nn + kK - 1) / kK, kh = (cols + kK - 1) / kK;
    ncta = grid;
    rw = tw / ncta, lw = tw % ncta;
    rh = th / ncta, lh = th % ncta;
    line = (i64)lw * max(kw, kEnd) + (i64)lh * max(kh, kEnd);
  }
  // What is left over: tile i of the line starts at...  It is as long as its
  // steps, or kEnd if they are fewer.  (Without that, 22 tiles of one step went to
  // one pair beside others' 21 steps of a long one: 64 tokens, 113 us and not 44.)
  OSSM_DEV i64 start(int i) const {
    return i < lw ? (i64)i * max(kw, kEnd) : (i64)lw * max(kw, kEnd) + (i64)(i - lw) * max(kh, kEnd);
  }
  OSSM_DEV int steps(int i) const { return i < lw ? kw : kh; }
  OSSM_DEV int at(i64 pos) const {
    const i64 w = (i64)lw * max(kw, kEnd);
    return pos < w ? (int)(pos / max(kw, kEnd)) : lw + (int)((pos - w) / max(kh, kEnd));
  }
  // Where pair c's part of the line begins.  A cut within 16 steps of its tile's
  // edge (an eighth of a short one) moves to the edge.
  OSSM_DEV i64 cut(int c) const {
    if (c >= ncta) return line;
    const i64 pos = line / ncta * c + line % ncta * c / ncta;
    const int i = at(pos), k = steps(i), near = min(16, k / 8);
    const i64 s = start(i);
    return pos - s <= near ? s : pos - s >= k - near ? s + max(k, kEnd) : pos;
  }
};
struct Item {
  bool w;       // of dW
  int m0, n0;   // the tile
  int k0, k1;   // its steps here
  bool split;
  int rest;     // split: the tile's place on the line
};
struct Shares {  // of one pair, in order
  const Tiles& t;
  int cta, round;
  i64 pos, end;
  OSSM_DEV Shares(const Tiles& tiles, int c) : t(tiles), cta(c), round(0), pos(tiles.cut(c)), end(tiles.cut(c + 1)) {}
  OSSM_DEV bool next(Item& x) {
    int u;
    if (round < t.rw + t.rh) {
      x.w = round < t.rw;
      u = (x.w ? round : round - t.rw) * t.ncta + cta;
      ++round;
      x.k0 = 0, x.k1 = x.w ? t.kw : t.kh;
      x.split = false;
    } else {
      if (pos >= end) return false;
      const int i = t.at(pos);
      const i64 s = t.start(i);
      x.w = i < t.lw;
      u = x.w ? t.rw * t.ncta + i : t.rh * t.ncta + i - t.lw;
      x.k0 = (int)(pos - s);
      x.k1 = (int)min((i64)t.steps(i), end - s);
      x.split = x.k1 - x.k0 < t.steps(i);
      x.rest = i;
      pos = x.k1 == t.steps(i) ? s + max(x.k1, kEnd) : end;
    }
    x.m0 = u / t.nt * kM, x.n0 = u % t.nt * kN;
    return true;
  }
};
constexpr size_t kPart = (size_t)kHalf * kN;  // floats of a CTA's half of a tile's sums

// What becomes of a row's sums of a tile, 8 columns at a time.
template <typename T>
struct Finish {
  const Params& p;
  T* to;            // where the row's columns of this half go, or NULL
  float4* sum;      // dH's sums over the pieces of the vocabulary; float4 e of every row side by side
  int left;         // columns of this half that exist
  float unit;
  OSSM_DEV Finish(const Params& q, bool w, int tile, int rank, int row, int half, int r, int n, int cols, int n0)
      : p(q), to(nullptr), sum(nullptr), left(q.d - n0), unit(q.head->unit) {
    if (w) {
      if (r < cols) to = static_cast<T*>(p.dw) + (i64)(p.v0 + r) * p.d + n0;
    } else {
      if (r < n) to = static_cast<T*>(p.dh) + (i64)__ldg(p.rows + r) * p.d + n0;
      sum = reinterpret_cast<float4*>(p.dh32 + (2 * tile + rank) * kPart) + half * 32 * kHalf + row;
    }
  }
  OSSM_DEV bool out() const { return !sum || p.last; }  // they are outputs
  OSSM_DEV uint4 value(int e, const float* y) const {    // columns 8 e .. 8 e + 7, as outputs
    float4 a = make_float4(y[0], y[1], y[2], y[3]), b = make_float4(y[4], y[5], y[6], y[7]);
    if (8 * e >= left) return make_uint4(0, 0, 0, 0);
    if (sum && !p.first) {
      const float4 u = sum[2 * e * kHalf], v = sum[(2 * e + 1) * kHalf];
      a.x += u.x, a.y += u.y, a.z += u.z, a.w += u.w;
      b.x += v.x, b.y += v.y, b.z += v.z, b.w += v.w;
    }
    if (!out()) sum[2 * e * kHalf] = a, sum[(2 * e + 1) * kHalf] = b;
    return make_uint4(pack2<T>(a.x * unit, a.y * unit), pack2<T>(a.z * unit, a.w * unit),
                      pack2<T>(b.x * unit, b.y * unit), pack2<T>(b.z * unit, b.w * unit));
  }
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    lce_prod_kernel(const __grid_constant__ CUtensorMap mZm, const __grid_constant__ CUtensorMap mZk,
                    const __grid_constant__ CUtensorMap mH, const __grid_constant__ CUtensorMap mHc,
                    const __grid_constant__ CUtensorMap mW, const __grid_constant__ Params p) {
  constexpr int S = kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Shared<S> s;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = cluster_rank(), pair = blockIdx.x >> 1;
  setup(s, warp);
  const int n = p.head->n, cols = min(p.vp, p.V - p.v0);
  const Tiles tiles(p, n, cols, gridDim.x >> 1);
  Shares todo(tiles, pair);
  Item x;

  if (warp == 8) {
    if (lane == 0) {
      const CUtensorMap* hm = n == p.T ? &mH : &mHc;
      Loader<S> ld{s, smem, rank == 0, 0, 0, 0};
      bool ok = true;
      while (ok && todo.next(x)) {
        const int boxes = p.d - x.n0 > 128 ? 2 : 1;  // a CTA's share of the tile's 256 or 128 columns
        const int m0 = x.m0 + rank * kHalf, n0 = x.n0 + rank * boxes * 64;
        for (int k = x.k0; k < x.k1; ++k) {
          uint32_t bar;
          uint8_t* to = ld.next(kABytes + boxes * kBox, bar);
          if (!to) {
            ok = false;
            break;
          }
          if (x.w) {
            tma_load_2d(to, &mZm, bar, m0, k * kK);
            tma_load_2d(to + kBox, &mZm, bar, m0 + 64, k * kK);
            for (int i = 0; i < boxes; ++i) tma_load_2d(to + kABytes + i * kBox, hm, bar, n0 + 64 * i, k * kK);
          } else {
            tma_load_2d(to, &mZk, bar, k * kK, m0);
            for (int i = 0; i < boxes; ++i)
              tma_load_2d(to + kABytes + i * kBox, &mW, bar, n0 + 64 * i, p.v0 + k * kK);
          }
        }
      }
      ld.end(ok);
    }
  } else if (warp == 9) {
    if (rank == 0) {
      const bool leader = elect_one();
      constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
      Issuer<S> mm{s, smem_u32(smem), 0, 0, 0};
      bool ok = true;
      while (ok && todo.next(x))
        ok = mm.tile(x.k1 - x.k0, idesc(fmt, x.w, 1, p.d - x.n0 > 128 ? 256 : 128), x.w ? 2048 : 32, 2048, leader);
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tl = s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 128;
    const uint32_t freed[2] = {first_cta(&s.acc_empty[0]), first_cta(&s.acc_empty[1])};
    uint8_t* const box = smem + S * kStage + warp * 2048;  // 32 rows x 32 columns
    uint32_t done = 0;
    bool dead = false;
    for (; todo.next(x); ++done) {
      const uint32_t b = done & 1;
      if (!dead) dead = gave_up(&s.acc_full[b], (done >> 1) & 1, &s.failed);
      __syncwarp();
      tc_fence_after();
      const int r = x.m0 + rank * kHalf + row, n0 = x.n0 + half * 128;
      const Finish<T> fin(p, x.w, x.m0 / kM * tiles.nt + x.n0 / kN, rank, row, half, r, n, cols, n0);
      float4* part = reinterpret_cast<float4*>(p.cuts + (2 * blockIdx.x + (x.k0 == 0)) * kPart) + half * 32 * kHalf + row;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        if (n0 + 32 * i >= p.d) break;
        float y[32];
        tmem_ld32_nowait(tl + b * kN + 32 * i, y);
        tmem_wait_ld();
        pin32(y);
        if (x.split) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            part[(8 * i + e) * kHalf] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
        } else {
          // outputs by way of shared memory, so that a store has whole sectors (16 bytes of 32 rows each
          // kept the tiles of a short product, 64 tokens and 50000 columns, at 0.6 TB/s)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 v = fin.value(4 * i + e, y + 8 * e);
            *reinterpret_cast<uint4*>(box + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) = v;
          }
          __syncwarp();
          if (fin.out()) {
            const int c = lane & 3;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int q = 8 * k + (lane >> 2);
              T* const at = reinterpret_cast<T*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(fin.to), q));
              const uint4 v = *reinterpret_cast<const uint4*>(box + q * 64 + ((c ^ ((q >> 1) & 3)) << 4));
              if (at && 32 * i + 8 * c < fin.left) *reinterpret_cast<uint4*>(at + 32 * i + 8 * c) = v;
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(freed[b]);
    }
  }
  teardown(s, warp, p.status);
}

// The tiles that were cut: blocks (.., c) take the one that pair c + 1's part
// begins in, if no earlier part begins there; a block adds up 32 columns of 128
// rows of it, a thread 8 columns of a row, 4 pieces on their way.
constexpr int kJoinThreads = 4 * kHalf, kMaxPairs = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 2) lce_join_kernel(const __grid_constant__ Params p, int pairs) {
  const int n = p.head->n, cols = min(p.vp, p.V - p.v0);
  const Tiles t(p, n, cols, pairs);
  const int rank = blockIdx.x & 1, half = blockIdx.x >> 1 & 1, row = threadIdx.x % kHalf;
  const int e = 4 * (blockIdx.x >> 2) + threadIdx.x / kHalf;
  __shared__ i64 cuts[kMaxPairs + 1];
  for (int c = threadIdx.x; c <= pairs; c += kJoinThreads) cuts[c] = t.cut(c);
  __syncthreads();
  const i64 begin = cuts[blockIdx.y + 1];
  if (begin >= t.line) return;
  const int i = t.at(begin);
  const i64 from = t.start(i), upto = from + t.steps(i);
  if (begin == from || cuts[blockIdx.y] > from) return;  // no cut, or not its first
  const bool w = i < t.lw;
  const int u = w ? t.rw * t.ncta + i : t.rh * t.ncta + i - t.lw;
  const int m0 = u / t.nt * kM, n0 = u % t.nt * kN + half * 128;
  // from the pair in whose part the tile starts to the one where it ends
  const int c0 = blockIdx.y;
  int c1 = c0 + 1;
  while (cuts[c1] < upto) ++c1;
  const int r = m0 + rank * kHalf + row;
  const Finish<T> fin(p, w, m0 / kM * t.nt + u % t.nt, rank, row, half, r, n, cols, n0);
  if (n0 + 8 * e >= p.d) return;
  float y[8] = {};
  const float4* q = reinterpret_cast<const float4*>(p.cuts) + (half * 32 + 2 * e) * kHalf + row;
  for (int c = c0; c < c1; c += 4) {
    float4 a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = c + k < c1 && (c + k == c0 || cuts[c + k + 1] > cuts[c + k]);  // has a part at all
      const float4* v = q + (4 * (i64)(c + k) + 2 * rank + (c + k == c0)) * (kPart / 4);
      a[k] = in ? __ldg(v) : make_float4(0.f, 0.f, 0.f, 0.f);
      b[k] = in ? __ldg(v + kHalf) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[0] += a[k].x, y[1] += a[k].y, y[2] += a[k].z, y[3] += a[k].w;
      y[4] += b[k].x, y[5] += b[k].y, y[6] += b[k].z, y[7] += b[k].w;
    }
  }
  const uint4 v = fin.value(e, y);
  if (fin.out() && fin.to) *reinterpret_cast<uint4*>(fin.to + 8 * e) = v;
}

// ---------------------------------------------------------------- rows
template <int THREADS, typename V, typename F>
OSSM_DEV V block_reduce(V v, V* warps, F f) {  // of a block's threads, the same in all of them
#pragma unroll
  for (int w = 16; w; w >>= 1) v = f(v, __shfl_xor_sync(~0u, v, w));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  v = warps[threadIdx.x % (THREADS / 32)];
#pragma unroll
  for (int w = THREADS / 64; w; w >>= 1) v = f(v, __shfl_xor_sync(~0u, v, w));
  return v;
}

// Which tokens have a target: their numbers in order, their targets, and, if
// some have none, their states side by side.  Backward: the factors of each
// row's gradient, zeros in dH where there is no target.  Every block counts
// the tokens before its own (they are in L2), so that none waits for another.
template <bool BWD>
__global__ void __launch_bounds__(kRowThreads) lce_rows_kernel(const __grid_constant__ Params p) {
  __shared__ i64 wi[kRowThreads / 32];
  __shared__ float wf[kRowThreads / 32];
  __shared__ int places[kRowThreads], total[kRowThreads / 32];
  const i64 chunk = (p.T + gridDim.x - 1) / gridDim.x, c0 = min(p.T, chunk * blockIdx.x), c1 = min(p.T, c0 + chunk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  i64 before = 0, all = 0;
  float top = 0.f;
  for (i64 t0 = threadIdx.x; t0 < p.T; t0 += 8 * kRowThreads) {  // 8 loads on their way
    bool has[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const i64 t = t0 + i * kRowThreads;
      has[i] = t < p.T && __ldg(p.targets + t) != p.ignore;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      all += has[i];
      before += has[i] && t0 + i * kRowThreads < c0;
    }
    if (BWD && (p.zl > 0.f || !p.reduction)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const i64 t = t0 + i * kRowThreads;
        const float f = p.reduction || t >= p.T ? 1.f : fabsf(__ldg(p.g + t));
        const float l = p.zl > 0.f && t < p.T ? __ldg(p.lse + t) : 0.f;
        const float factor = f * fmaxf(1.f, fabsf(1.f + 2.f * p.zl * l));
        if (has[i] && isfinite(factor)) top = fmaxf(top, factor);  // others spoil their own row alone
      }
    } else if (BWD) {
      top = 1.f;
    }
  }
  auto plus = [](i64 a, i64 b) { return a + b; };
  all = block_reduce<kRowThreads>(all, wi, plus);
  before = block_reduce<kRowThreads>(before, wi, plus);
  const int n = (int)all;
  float scale = 1.f;
  if (BWD) {
    top = block_reduce<kRowThreads>(top, wf, [](float a, float b) { return fmaxf(a, b); });
    if (p.reduction) scale = __ldg(p.g) / (p.reduction == 1 ? (float)max(n, 1) : 1.f);
  }
  const float inv = top > 0.f ? fminf(kDzScale / top, 0x1p120f) : 0.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.head->n = n;
    p.head->unit = inv > 0.f ? scale / inv : 0.f;
    p.head->count = 0;
  }
  const bool gather = all < p.T;
  const int vecs = p.d / 8;
  i64 base = before;
  for (i64 t0 = c0; t0 < c1; t0 += kRowThreads) {
    const i64 t = t0 + threadIdx.x;
    const i64 target = t < c1 ? __ldg(p.targets + t) : 0;
    const bool has = t < c1 && target != p.ignore;
    const uint32_t votes = __ballot_sync(~0u, has);
    __syncthreads();
    if (lane == 0) total[warp] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1)), count = 0;
    for (int i = 0; i < kRowThreads / 32; ++i) {
      if (i < warp) at += total[i];
      count += total[i];
    }
    const i64 place = base + at;
    base += count;
    places[threadIdx.x] = has ? (int)place : -1;
    const bool known = target >= 0 && target < p.V;
    if (has) {
      p.rows[place] = (int)t;
      p.tgt[place] = known ? (int)target : -1;
      if (BWD) {
        const float lse = __ldg(p.lse + t), g = p.reduction ? 1.f : __ldg(p.g + t);
        // a target outside the vocabulary: NaN, as its loss
        const float f = known ? g * inv : NAN;
        // the exponent takes lse in fp32, its factor what that leaves: a sure token's
        // gradient is the difference of a probability and 1
        const double l2 = ((double)lse + (p.rest ? (double)__ldg(p.rest + t) : 0.0)) * 1.4426950408889634;
        const float hi = (float)l2, left = (float)((double)hi - l2);
        p.lse2[place] = hi;
        p.fa[place] = f * (1.f + 2.f * p.zl * lse) * (fabsf(left) < 1.f ? fmaf(left, 0.6931472f, 1.f) : 1.f);
        p.fb[place] = f;
      }
    } else if (!BWD && t < c1) {
      p.lse[t] = 0.f;
      if (p.rest) p.rest[t] = 0.f;
      if (!p.reduction) p.loss[t] = 0.f;
    }
    if (!gather) continue;
    __syncthreads();
    const int count_here = (int)min((i64)kRowThreads, c1 - t0), pieces = count_here * vecs;
    for (int e0 = threadIdx.x; e0 < pieces; e0 += 8 * kRowThreads) {
      uint4 v[8];
      int row[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = e0 + k * kRowThreads;
        row[k] = e / vecs;
        if (e < pieces && places[row[k]] >= 0)
          v[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.hidden) + (t0 + row[k]) * p.hst) +
                       (e - row[k] * vecs));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = e0 + k * kRowThreads, at = e - row[k] * vecs;
        if (e >= pieces) break;
        const int to = places[row[k]];
        if (to >= 0)
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.hc) + (i64)to * p.dst)[at] = v[k];
        else if (BWD && p.dh)
          reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dh) + (t0 + row[k]) * p.d)[at] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (gather && blockIdx.x == gridDim.x - 1) {  // the last block of rows is read whole
    const int to = (max(n, 1) + kM - 1) / kM * kM;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.hc) + (i64)n * p.dst);
    for (i64 e = threadIdx.x; e < (i64)(to - n) * (p.dst / 8); e += kRowThreads) dst[e] = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------- losses
// 2 to 32 lanes a row join the partial sums, by their number; block sums in
// float64, added in order by the last block.
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads) lce_finish_kernel(const __grid_constant__ Params p, const int lanes) {
  __shared__ double ws[kFinishThreads / 32];
  __shared__ bool last;
  const int n = p.head->n, mine = threadIdx.x & (lanes - 1), per = kFinishThreads / lanes;
  double sum = 0.0;
  for (int r0 = blockIdx.x * per; r0 < n; r0 += gridDim.x * per) {
    const int r = r0 + threadIdx.x / lanes;
    float m = -INFINITY, l = 0.f;
    if (r < n) {
      const float2* q = p.part + (i64)r * 2 * p.panels;
      for (int i0 = mine; i0 < 2 * p.panels; i0 += 8 * lanes) {
        float2 v[8];
        float top = m;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = i0 + k * lanes < 2 * p.panels ? __ldg(q + i0 + k * lanes) : make_float2(-INFINITY, 0.f);
          top = fmaxf(top, v[k].x);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        l *= ex2(m - ref);
#pragma unroll
        for (int k = 0; k < 8; ++k) l = fmaf(v[k].y, ex2(v[k].x - ref), l);
        m = top;
      }
    }
    for (int w = lanes >> 1; w; w >>= 1) {
      const float m2 = __shfl_xor_sync(~0u, m, w), l2 = __shfl_xor_sync(~0u, l, w);
      const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
      l = l * ex2(m - ref) + l2 * ex2(m2 - ref);
      m = top;
    }
    if (r < n && mine == 0) {
      const int t = p.rows[r];
      const double lse2 = (double)m + log2((double)l), lse = lse2 * 0.6931471805599453;
      // less the target's logit in the same units: log2(e) is kLog2e in both
      double loss = (lse2 - (double)p.zt[r] * (double)kLog2e) * 0.6931471805599453 + (double)p.zl * lse * lse;
      if (p.tgt[r] < 0) loss = NAN;
      p.lse[t] = (float)lse;
      if (p.rest) p.rest[t] = isfinite(lse) ? (float)(lse - (double)(float)lse) : 0.f;
      if (!p.reduction) p.loss[t] = (float)loss;
      sum += loss;
    }
  }
  if (!p.reduction) return;
  auto plus = [](double a, double b) { return a + b; };
  sum = block_reduce<kFinishThreads>(sum, ws, plus);
  if (threadIdx.x == 0) {
    p.sums[blockIdx.x] = sum;
    __threadfence();
    last = atomicAdd(&p.head->count, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double all = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kFinishThreads) all += __ldcg(p.sums + i);
  all = block_reduce<kFinishThreads>(all, ws, plus);
  if (threadIdx.x == 0) *p.loss = (float)(p.reduction == 1 ? all / max(n, 1) : all);
}

// ---------------------------------------------------------------- host
bool valid(const ossm_lce_args* a, bool bwd) {
  if (!a || a->tokens < 1 || a->tokens > (1 << 27) || a->vocab < 1 || a->vocab > (1 << 27)) return false;
  if (a->dim < 8 || a->dim % 8 || a->dim > (1 << 16)) return false;
  if (a->dtype != OSSM_BF16 && a->dtype != OSSM_F16) return false;
  if (a->reduction < OSSM_LOSS_NONE || a->reduction > OSSM_LOSS_SUM) return false;
  if (!(a->z_loss >= 0.f) || !std::isfinite(a->z_loss)) return false;
  auto rows_ok = [&](const void* q, i64 st) { return q && (uintptr_t)q % 16 == 0 && st % 8 == 0 && st >= a->dim; };
  if (!rows_ok(a->hidden, a->hidden_stride) || !rows_ok(a->weight, a->weight_stride)) return false;
  if (!a->targets || !a->lse) return false;
  if (!bwd) return a->loss != nullptr;
  return a->grad_loss && (uintptr_t)a->grad_hidden % 16 == 0 && (uintptr_t)a->grad_weight % 16 == 0;
}

struct Plan {
  int Tpad, Vpad, sms, ntiles, pan, panels, vp;
  size_t at[12], bytes;
};
// The workspace, and how the vocabulary is cut.
Plan plan_of(const ossm_lce_args* a, bool bwd) {
  Plan q{};
  q.sms = std::min(device_sms(), 2 * kMaxPairs) & ~1;
  q.Tpad = (int)((a->tokens + 255) / 256 * 256);
  q.Vpad = (a->vocab + kN - 1) / kN * kN;
  const i64 blocks = (a->tokens + kM - 1) / kM, pairs = q.sms / 2;
  // Backward: dZ of a piece takes at most 512 MB, but has 4096 columns at
  // least: each piece reads and writes dH's fp32 sums once.
  q.vp = bwd ? (int)std::min<i64>(q.Vpad, std::max<i64>(4096, (1LL << 28) / q.Tpad / kN * kN)) : q.Vpad;
  q.ntiles = q.vp / kN;
  // A row's sums stay in registers over a panel: up to 8 tiles, fewer where
  // there would not be 6 panels for each pair to even out.
  q.pan = bwd ? 1 : (int)std::min<i64>(8, std::max<i64>(1, blocks * q.ntiles / (6 * pairs)));
  q.panels = (q.ntiles + q.pan - 1) / q.pan;
  size_t at = 0;
  int k = 0;
  auto take = [&](size_t bytes) {
    q.at[k++] = at;
    at += (bytes + 255) / 256 * 256;
  };
  const size_t T = q.Tpad, d = a->dim;
  take(sizeof(Head));
  take(4 * T);              // rows
  take(4 * T);              // targets
  take(2 * T * ((d + 63) / 64 * 64));  // states side by side
  if (!bwd) {
    take(8 * T * 2 * q.panels);
    take(4 * T);
    take(8 * kMaxBlocks);
  } else {
    take(4 * T);
    take(4 * T);
    take(4 * T);
    take(2 * T * (size_t)q.vp);  // dz
    const size_t nt = (d + kN - 1) / kN;
    take(a->grad_hidden && q.vp < q.Vpad ? 4 * T * nt * kN : 0);
    take(2 * q.sms * kPart * 4);
  }
  q.bytes = at;
  return q;
}

// [rows, inner] with 128-byte swizzle, box [brows, 64].
bool encode(CUtensorMap* map, int dtype, const void* base, i64 inner, i64 rows, i64 stride, int brows) {
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)brows}, estr[2] = {1, 1};
  return fast::encode_fn()(map, dtype == OSSM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Params params_of(const ossm_lce_args* a, const Plan& q, char* w, bool bwd) {
  Params p{};
  p.T = a->tokens, p.Tpad = q.Tpad, p.d = a->dim, p.V = a->vocab;
  p.dst = (a->dim + 63) / 64 * 64;
  p.hidden = a->hidden, p.hst = a->hidden_stride;
  p.targets = a->targets, p.ignore = a->ignore_index, p.zl = a->z_loss, p.reduction = a->reduction;
  p.loss = a->loss, p.lse = a->lse, p.rest = a->lse_rest, p.g = a->grad_loss, p.dh = a->grad_hidden, p.dw = a->grad_weight;
  p.head = reinterpret_cast<Head*>(w + q.at[0]);
  p.rows = reinterpret_cast<int*>(w + q.at[1]);
  p.tgt = reinterpret_cast<int*>(w + q.at[2]);
  p.hc = w + q.at[3];
  if (!bwd) {
    p.part = reinterpret_cast<float2*>(w + q.at[4]);
    p.zt = reinterpret_cast<float*>(w + q.at[5]);
    p.sums = reinterpret_cast<double*>(w + q.at[6]);
  } else {
    p.lse2 = reinterpret_cast<float*>(w + q.at[4]);
    p.fa = reinterpret_cast<float*>(w + q.at[5]);
    p.fb = reinterpret_cast<float*>(w + q.at[6]);
    p.dh32 = reinterpret_cast<float*>(w + q.at[8]);
    p.cuts = reinterpret_cast<float*>(w + q.at[9]);
  }
  p.panels = q.panels, p.pan = q.pan, p.vp = q.vp;
  p.status = a->status;
  return p;
}

// A block for 32 tokens, up to one an SM.
int row_blocks(const Plan& q, i64 T) { return (int)std::min<i64>(q.sms, (T + 31) / 32); }

template <typename T>
int forward(const ossm_lce_args* a, const Plan& q, char* w, cudaStream_t st) {
  Params p = params_of(a, q, w, false);
  CUtensorMap mh, mc, mw;
  if (!encode(&mh, a->dtype, a->hidden, a->dim, a->tokens, a->hidden_stride, kHalf) ||
      !encode(&mc, a->dtype, p.hc, a->dim, q.Tpad, p.dst, kHalf) ||
      !encode(&mw, a->dtype, a->weight, a->dim, a->vocab, a->weight_stride, kHalf))
    return OSSM_EINVAL;
  lce_rows_kernel<false><<<row_blocks(q, a->tokens), kRowThreads, 0, st>>>(p);
  static std::atomic<uint64_t> done{0};
  auto kern = lce_logits_kernel<T, STATS>;
  constexpr size_t smem = smem_bytes(kStages, 0);
  if (allow_smem(kern, (int)smem, done) != cudaSuccess) return OSSM_ELAUNCH;
  const i64 items = (a->tokens + kM - 1) / kM * q.panels;
  kern<<<(int)std::min<i64>(q.sms, 2 * items), kThreads, smem, st>>>(mh, mc, mw, mw, p);
  int lanes = 2;
  while (lanes < 32 && lanes * 8 < 2 * q.panels) lanes *= 2;
  const int blocks = (int)std::min<i64>(kMaxBlocks, (a->tokens * lanes + kFinishThreads - 1) / kFinishThreads);
  lce_finish_kernel<<<blocks, kFinishThreads, 0, st>>>(p, lanes);
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

template <typename T>
int backward(const ossm_lce_args* a, const Plan& q, char* w, cudaStream_t st) {
  Params p = params_of(a, q, w, true);
  void* dz = w + q.at[7];
  CUtensorMap mh, mc, mw, ms, mzm, mzk, hm, hcm, wm;
  if (!encode(&mh, a->dtype, a->hidden, a->dim, a->tokens, a->hidden_stride, kHalf) ||
      !encode(&mc, a->dtype, p.hc, a->dim, q.Tpad, p.dst, kHalf) ||
      !encode(&mw, a->dtype, a->weight, a->dim, a->vocab, a->weight_stride, kHalf) ||
      !encode(&ms, a->dtype, dz, q.vp, q.Tpad, q.vp, 32) || !encode(&mzm, a->dtype, dz, q.vp, q.Tpad, q.vp, 64) ||
      !encode(&mzk, a->dtype, dz, q.vp, q.Tpad, q.vp, kHalf) ||
      !encode(&hm, a->dtype, a->hidden, a->dim, a->tokens, a->hidden_stride, 64) ||
      !encode(&hcm, a->dtype, p.hc, a->dim, q.Tpad, p.dst, 64) ||
      !encode(&wm, a->dtype, a->weight, a->dim, a->vocab, a->weight_stride, 64))
    return OSSM_EINVAL;
  lce_rows_kernel<true><<<row_blocks(q, a->tokens), kRowThreads, 0, st>>>(p);
  static std::atomic<uint64_t> done_z{0}, done_p{0};
  auto gradz = lce_logits_kernel<T, GRADZ>;
  auto prod = lce_prod_kernel<T>;
  constexpr size_t smem_z = smem_bytes(kStagesZ, kOutZ), smem_p = smem_bytes(kStages, kOutP);
  if (allow_smem(gradz, (int)smem_z, done_z) != cudaSuccess || allow_smem(prod, (int)smem_p, done_p) != cudaSuccess)
    return OSSM_ELAUNCH;
  for (int v0 = 0; v0 < a->vocab; v0 += q.vp) {
    p.v0 = v0, p.first = v0 == 0, p.last = v0 + q.vp >= a->vocab;
    gradz<<<q.sms, kThreads, smem_z, st>>>(mh, mc, mw, ms, p);
    prod<<<q.sms, kThreads, smem_p, st>>>(mzm, mzk, hm, hcm, wm, p);
    lce_join_kernel<T><<<dim3(16, q.sms / 2 - 1), kJoinThreads, 0, st>>>(p, q.sms / 2);
  }
  return cudaGetLastError() == cudaSuccess ? OSSM_OK : OSSM_ELAUNCH;
}

}  // namespace lce
}  // namespace ossm

using namespace ossm;

extern "C" size_t ossm_lce_workspace_bytes(const ossm_lce_args* a, int backward) {
  return lce::valid(a, backward != 0) ? lce::plan_of(a, backward != 0).bytes : 0;
}

static int lce_call(const ossm_lce_args* a, void* workspace, size_t bytes, ossm_stream_t stream, bool bwd) {
  if (!lce::valid(a, bwd)) return OSSM_EINVAL;
  const lce::Plan q = lce::plan_of(a, bwd);
  if (!workspace || bytes < q.bytes || (uintptr_t)workspace % 256) return OSSM_EWORKSPACE;
  if (bwd && !a->grad_hidden && !a->grad_weight) return OSSM_OK;
  if (!fast::encode_fn()) return OSSM_ELAUNCH;
  char* w = static_cast<char*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a->dtype == OSSM_BF16;
  if (bwd) return bf ? lce::backward<__nv_bfloat16>(a, q, w, st) : lce::backward<__half>(a, q, w, st);
  return bf ? lce::forward<__nv_bfloat16>(a, q, w, st) : lce::forward<__half>(a, q, w, st);
}

extern "C" int ossm_lce_fwd(const ossm_lce_args* a, void* workspace, size_t workspace_bytes, ossm_stream_t stream) {
  return lce_call(a, workspace, workspace_bytes, stream, false);
}
extern "C" int ossm_lce_bwd(const ossm_lce_args* a, void* workspace, size_t workspace_bytes, ossm_stream_t stream) {
  return lce_call(a, workspace, workspace_bytes, stream, true);
}
extern "C" size_t ossm_sizeof_lce_args(void) { return sizeof(ossm_lce_args); }
