// attention_tc.cu -- attention of many query rows per key/value head (prompts,
// a shared prefix) over the paged cache, on the 5th-generation tensor cores.
//
// An item is QT tiles of 128 query rows (attention.cuh: the heads of a group
// share their keys, so 8 heads make a tile of 16 tokens); QT = 2, or 1 above
// head size 128, where O takes half of TMEM.  Per tile of 64 keys and query
// tile: S = Q K^T into one of two S buffers in TMEM, two softmax threads per
// row with 32 keys each, P as bf16 back over S, O += P V with P as the TMEM
// operand and V in its natural token-major layout (MN-major operand).  The next
// S is issued before the product that waits for P, so a softmax finds its next
// S ready and its warps never stop; O stays in TMEM for all of an item.
//   warps 0-7 (and 8-15, QT = 2)  softmax of tile 0 (1), Q into shared memory,
//                                 the rare rescaling of O, the epilogue;
//   then one warp each            MMA issue for each query tile, TMA producer,
//                                 and the block's list of items with the
//                                 zeroing of values that no row sees.
// O is rescaled only when a row's maximum has grown by more than 2^8 since
// the last time (weights then stay below 2^8, exact in the sums' fp32); the
// reference is the same for sum and product, so the result is not changed.
// A row's two threads meet once per tile, to learn whether either saw such a
// growth.  (One thread per row: 19 us more of 278, four ragged prompts at head
// size 256, where a tile's softmax is the one in flight; 572 against 570 us for a
// prompt of 8192 at 32 / 4 heads of 128.)
//
// What bounds it: that prompt takes 548 to 574 us, 960 to 1000 TFLOP/s, at 990 W,
// where the power limit takes the clock from 1965 to 1680 MHz.  Per pair of query tiles and key
// tile it takes 1950 cycles: the exponentials 1024 of the MUFU, in a phase of
// all warps that nothing else fills, and the products 1050 of the tensor cores.
// Exponentials on the FMA pipe in part (a polynomial of degree 4) give 587 to
// 620 us from 1/8 to 1/2 of them, the exponentials of the two query tiles taken
// in turns 597: more instructions at the same power.  Head size 256 loads 64 KB
// per tile of 128 rows and is bound by that: those ragged prompts, in pages of 16,
// take 235 us, 720 TFLOP/s (277 while a copy brought 64 of a value's columns; 213
// without the output gate).
#include <cuda_bf16.h>

#include <type_traits>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention.cuh"
#include "attention_launch.h"
#include "kernels.h"
#include "tc_common.cuh"

namespace nvfp4 {

static __device__ int g_attn_tc_status;

namespace {

constexpr int kSegs = 4;      // items that the scheduling warp may be ahead

constexpr int KT = 64;        // keys per tile
constexpr int HK = KT / 2;    // of them a softmax thread's

// Of an item's beginning and end, in key tiles, which two query tiles with capped
// or biased scores take longer for.  (A prompt of 8192, 32 / 4 heads of 128: 618 us
// with 2, 569 with 5, 569 with 8.  Four ragged ones at head size 256: 245 with 2,
// 235 with 5, 236 with 8.  Capped or biased, with 2, 3 and 5: three prompts of 28 / 4
// heads of 128 146, 147 and 153 us, without bias and window 137, 135 and 142, of 8 / 8
// heads of 64 64, 66 and 69, the prompt of 8192 942, 946 and 960, the four with bias at
// head size 128 298, 290 and 285; at head size 256 the three 123, 123 and 126, the
// four 268, 262 and 258.)
template <int DP, bool MOD>
constexpr int kItemCost = MOD && DP <= 128 ? 2 : 5;

template <int DP>
struct TcCfg {
  static constexpr int QT = DP <= 128 ? 2 : 1;
  static constexpr int R = 128 * QT;
  static constexpr int kTile = KT * DP * 2;         // bytes of a key or value tile
  static constexpr int kQ = 128 * DP * 2;           // bytes of a query tile
  static constexpr int kSlots = DP == 64 ? 16 : DP == 128 ? 9 : 4;
  static constexpr int kSoftWarps = 8 * QT;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;
  static constexpr int offKV = QT * kQ;
  static constexpr int bytes = offKV + kSlots * kTile + 1024;
  // TMEM columns: two S buffers per query tile, then O of each.
  static constexpr int colO = 2 * QT * KT;
  static constexpr int cols = 512;
};

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 lanes x 32 columns: lane l gets columns 8 k + 2 (l % 4) + {0, 1} of rows
// l / 4 (r[4 k], r[4 k + 1]) and l / 4 + 8 (r[4 k + 2], r[4 k + 3]).
__device__ __forceinline__ void tmem_ld_16x256_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The warp that issues the MMAs runs as one, its operands the same in every
// lane (they belong in uniform registers).  Four k-steps of 16 go into one
// block of instructions, predicated on one elected lane without a branch
// around them: an operand that has to be made uniform for each MMA, or a
// branch, costs as much as the MMA takes the tensor cores.
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;  // 1024-byte groups, version, 128-byte swizzle

// D[tmem] (+)= A[smem] B[smem]^T over 64 columns; alo, blo: low words of the
// operands' descriptors, a k-step 32 bytes further along the swizzled rows.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t acc) {
#define NVFP4_SS_STEP(off, pred)                        \
  "add.u32 x, %1, " off ";\n\tadd.u32 y, %2, " off ";\n\t" \
  "mov.b64 ad, {x, %5};\n\tmov.b64 bd, {y, %5};\n\t"      \
  "@q tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, " pred ";\n\t"
  asm volatile(
      "{\n\t.reg .pred p, q, one;\n\t.reg .b32 x, y;\n\t.reg .b64 ad, bd;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 one, 0, 0;\n\t" NVFP4_SS_STEP("0", "p") NVFP4_SS_STEP("2", "one")
          NVFP4_SS_STEP("4", "one") NVFP4_SS_STEP("6", "one") "}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
#undef NVFP4_SS_STEP
}
// D[tmem] (+)= A[tmem] B[smem] over 64 tokens: 8 columns of A a k-step, and of B
// b1 (an odd step) and b2 (two steps) 16-byte units.
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, uint32_t acc, uint32_t b1,
                                        uint32_t b2) {
#define NVFP4_TS_STEP(aoff, boff, pred)                                  \
  "add.u32 x, %1, " aoff ";\n\t" boff "mov.b64 bd, {y, %5};\n\t" \
  "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], bd, %3, " pred ";\n\t"
  asm volatile(
      "{\n\t.reg .pred p, q, one;\n\t.reg .b32 x, y;\n\t.reg .b64 bd;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 one, 0, 0;\n\t" NVFP4_TS_STEP("0", "mov.b32 y, %2;\n\t", "p")
          NVFP4_TS_STEP("8", "add.u32 y, %2, %6;\n\t", "one") NVFP4_TS_STEP("16", "add.u32 y, %2, %7;\n\t", "one")
              NVFP4_TS_STEP("24", "add.u32 y, y, %6;\n\t", "one") "}" ::"r"(d),
      "r"(a), "r"(blo), "r"(idesc), "r"(acc), "r"(kDescHi), "r"(b1), "r"(b2)
      : "memory");
#undef NVFP4_TS_STEP
}
__device__ __forceinline__ void commit_to(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}

// Low word of a descriptor.  Keys and queries are K-major (the leading offset
// is not used, 16 bytes); values [token][d], 64 columns of 128 swizzled bytes
// per token, are an MN-major B operand: 64-column blocks (leading offset) and
// groups of 8 tokens 1024 bytes apart (stride offset).  A value tile lies box by
// box, each with its columns' blocks one after the other, as one copy of a box
// writes them; a key tile, block by block over all boxes, as one MMA reads it.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lead) {
  return ((saddr & 0x3FFFFu) >> 4) | (lead >> 4) << 16;
}
constexpr uint32_t kTransposeB = 1u << 16;

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Two fp32 at a time.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float &x, float &y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The largest of three.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

template <int DP, bool MOD>
__global__ void __launch_bounds__(TcCfg<DP>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ AttnArgs a) {
  using C = TcCfg<DP>;
  constexpr int QT = C::QT, R = C::R, kSlots = C::kSlots, E = kItemCost<DP, MOD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  __shared__ AttnPlanSmem plan;
  __shared__ uint64_t bars[3 * kSlots + 15 + 2 * kSegs];
  __shared__ AttnSegment segs[kSegs];
  __shared__ float row_x[2][R];  // a row's value of each of its two threads
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full = smem_u32(bars);
  const uint32_t empty = full + 8 * kSlots;   // the slot's MMAs are done
  const uint32_t edge = empty + 8 * kSlots;   // a value tile landed that needs zeroing
  const uint32_t bar_q = edge + 8 * kSlots;   // [2] queries of tile t in shared memory
  // Of query tile t and the parity x of its key tiles' count: [2 t + x].  Two
  // of each, so that none has more than one phase outstanding.
  const uint32_t bar_s = bar_q + 16;          // S ready
  const uint32_t bar_p = bar_s + 32;          // P written (and O rescaled)
  const uint32_t bar_o = bar_p + 32;          // P V done
  const uint32_t bar_end = bar_o + 32;
  const uint32_t seg_full = bar_end + 8;      // [kSegs] the block's next items
  const uint32_t seg_empty = seg_full + 8 * kSegs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, QT);  // a warp per query tile
      mbar_init(edge + 8 * i, 1);
    }
    mbar_init(bar_q, 8);
    mbar_init(bar_q + 8, 8);
    for (int x = 0; x < 4; ++x) {
      mbar_init(bar_s + 8 * x, 1);
      mbar_init(bar_p + 8 * x, 8);
      mbar_init(bar_o + 8 * x, 1);
    }
    mbar_init(bar_end, QT);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(seg_full + 8 * i, 1);
      mbar_init(seg_empty + 8 * i, C::kSoftWarps + QT + 2);
    }
    mbar_fence_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  // TMEM is taken after the launches before have ended and before a launch
  // behind this one may start: neither can hold what this block waits for.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == C::kSoftWarps) {
    tmem_alloc(smem_u32(&tmem_slot), C::cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;");
  AttnCursor cur = attn_plan<R, KT, E, 0>(a, 2 + E, &plan, C::kSoftWarps + 2);
  const uint32_t tmem = tmem_slot;
  if (threadIdx.x == 0) a.meta[blockIdx.x].last_part = -1;
  volatile int *abort = &abort_flag;
  int *status = &g_attn_tc_status;
  AttnSegment g;
  // The next item of the block from the scheduling warp's ring (every lane
  // of the warp calls it; take < 0: no more).
  uint32_t nseg = 0;
  auto next_seg = [&]() -> bool {
    const uint32_t i = nseg % kSegs;
    if (!__all_sync(0xffffffffu, attn_wait(seg_full + 8 * i, (nseg / kSegs) & 1, status, kDevTimeoutDec, abort)))
      return false;
    g = segs[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(seg_empty + 8 * i);
    ++nseg;
    return g.take >= 0;
  };
  // Tiles of an item in use: the second one only with rows beyond 128.
  auto tiles = [&](const AttnSegment &x) { return QT == 2 && x.s.ql * a.G - x.rb * R > 128 ? 2 : 1; };

  if (warp < C::kSoftWarps) {
    if constexpr (QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int t = warp >> 3, half = warp >> 2 & 1, wq = warp & 3;  // tile, half of the keys, lane quarter
    const int my = t * 128 + wq * 32 + lane;           // row within the item
    const uint32_t lanes = static_cast<uint32_t>(32 * wq) << 16;
    const uint32_t tO = tmem + lanes + C::colO + t * DP;
    uint8_t *Q = smem + t * C::kQ;
    const float c2 = MOD ? 1.0f : a.scale * kLog2e;
    const uint64_t c22 = pair(c2, c2);

    // The two warps of 32 rows.  Both always make the same calls: a warp whose
    // wait ran out goes on with what there is until the next item.
    const uint32_t bar_pair = 1 + 4 * t + wq;
    auto pair_any = [&](bool x) -> bool {
      uint32_t r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
          "barrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(r)
          : "r"((uint32_t)x), "r"(bar_pair)
          : "memory");
      return r != 0;
    };
    auto pair_other = [&](float x) -> float {  // the other thread's, of this row
      row_x[half][my] = x;
      asm volatile("barrier.cta.sync %0, 64;" ::"r"(bar_pair) : "memory");
      return row_x[half ^ 1][my];
    };

    // This warp's 16 rows of the next item's Q, 16-byte chunks swizzled as the
    // MMA reads them; rows and columns beyond the item's or the head's are
    // zeros.  Started here, handed over in q_done().
    auto q_start = [&]() {
      const int row = g.rb * R + my;
      const __nv_bfloat16 *src = nullptr;
      if (row < g.s.ql * a.G) {
        const int i = div_pos(row, a.G);
        src = a.q + (int64_t)(g.s.tok0 + i) * a.q_ts + (int64_t)(g.h * a.G + row - i * a.G) * a.q_hs;
      }
      constexpr int CH = DP / 8, RPI = 32 / CH;  // chunks per row, rows per warp step
      const int c = lane % CH;
#pragma unroll 4
      for (int r0 = 0; r0 < 16; r0 += RPI) {
        const int r = 16 * half + r0 + lane / CH;
        const uint64_t p = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), r);
        const int rr = wq * 32 + r;
        const bool on = p != 0 && 8 * c < a.D;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         smem_u32(Q + (c >> 3) * (128 * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4))),
                     "l"(on ? p + 16 * c : reinterpret_cast<uint64_t>(a.q)), "r"(on ? 16 : 0)
                     : "memory");
      }
    };
    auto q_done = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 8 * t);
    };

    uint32_t n = 0;  // key tiles of this query tile so far
    bool ok = true, have = !pair_any(!next_seg());
    bool fetch = have && g.take > 0 && t < tiles(g);
    if (fetch) {
      q_start();
      q_done();
    }
    while (have) {
      const bool mine = t < tiles(g);
      const int take = g.take, slot = g.slot, j_first = (g.it.u0 + g.off) * KT;
      const int row = g.rb * R + my;
      const bool in = mine && row < g.s.ql * a.G;
      if (g.last_part >= 0 && threadIdx.x == 0) a.meta[blockIdx.x] = attn_meta<R>(a, g);
      AttnRow ar = attn_row(a, g.s, g.h, in ? row : 0);
      if (!in) ar.lo = ar.hi = 0;
      // The gate comes from HBM: into L2 under the item's tiles.
      if (a.gate && in && slot < 0 && !a.prefix_pass) {
        const __nv_bfloat16 *p = a.gate + ar.token * a.g_ts + ar.head * a.g_hs;
        for (int c = 64 * half; c < a.D; c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + c));
      }
      float m = -INFINITY, l = 0.0f;
      if (mine && take > 0) {
        // Keys that all rows of the warp see need no mask.
        const int lo_all = __reduce_max_sync(0xffffffffu, ar.lo), hi_all = __reduce_min_sync(0xffffffffu, ar.hi);
        const float slope = MOD && a.slopes ? a.slopes[ar.head] * kLog2e : 0.0f;
        const int pos = ar.pos - (a.prefix_pass ? 0 : a.prefix_len);
#pragma unroll 1
        for (int u = 0; u < take; ++u, ++n) {
          const int j0 = j_first + u * KT + half * HK;
          const uint32_t x = 2 * t + (n & 1);
          const uint32_t tS = tmem + lanes + x * KT;
          ok = attn_wait(bar_s + 8 * x, (n >> 1) & 1, status, kDevTimeoutAcc, abort) && ok;
          __syncwarp();
          tc_fence_after();
          uint32_t raw[HK];
          tmem_ld_32x32b_x32(tS + half * HK, raw);
          tmem_ld_wait();
          float s[HK];
#pragma unroll
          for (int c = 0; c < HK; ++c) s[c] = __uint_as_float(raw[c]);
          if constexpr (MOD) {
            if (a.softcap > 0.0f) {  // cap tanh(scale s / cap), base 2 (tanh_log2e, two at a time)
#pragma unroll
              for (int c = 0; c < HK; c += 2) {
                float x0, x1, q0, q1;
                unpair(mul2(mul2(pair(s[c], s[c + 1]), pair(a.scale, a.scale)), pair(a.inv_cap, a.inv_cap)), x0, x1);
                const uint64_t t = pair(hold(x0, kTanhMax), hold(x1, kTanhMax)), u = mul2(t, t);
                uint64_t p = pair(tanh_p(4), tanh_p(4)), q = pair(tanh_q(4), tanh_q(4));
#pragma unroll
                for (int k = 3; k >= 0; --k) {
                  p = fma2(p, u, pair(tanh_p(k), tanh_p(k)));
                  q = fma2(q, u, pair(tanh_q(k), tanh_q(k)));
                }
                unpair(q, q0, q1);
                p = mul2(mul2(mul2(t, p), pair(rcp(q0), rcp(q1))), pair(a.softcap, a.softcap));
                unpair(p, s[c], s[c + 1]);
              }
            } else {
#pragma unroll
              for (int c = 0; c < HK; ++c) s[c] *= a.scale * kLog2e;
            }
            if (a.slopes) {
              const float dist = (float)(pos - j0);  // a conversion per element would be on the MUFU, too
#pragma unroll
              for (int c = 0; c < HK; ++c) s[c] = fmaf(-slope, fabsf(dist - (float)c), s[c]);
            }
          }
          if (j0 < lo_all || j0 + HK > hi_all) {
            const int lo = ar.lo - j0, hi = ar.hi - j0;
#pragma unroll
            for (int c = 0; c < HK; ++c) s[c] = c >= lo && c < hi ? s[c] : -INFINITY;
          }
          float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int c = 4; c < HK - 4; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = max3(top[i], s[c + i], s[c + 4 + i]);
          top[0] = max3(top[0], s[HK - 4], s[HK - 3]);
          top[1] = max3(top[1], s[HK - 2], s[HK - 1]);
          float mx = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * c2;
          // (Behind this barrier both threads have read their S, and P may go over it.)
          if (pair_any(mx > m + 8.0f)) {
            mx = fmaxf(mx, pair_other(mx));
            const bool grow = mx > m + 8.0f;
            const float mn = grow ? mx : m;
            if (u > 0) {  // O of the tiles before, once they are all in
              const uint32_t y = 2 * t + ((n - 1) & 1);
              ok = attn_wait(bar_o + 8 * y, ((n - 1) >> 1) & 1, status, kDevTimeoutAcc, abort) && ok;
              __syncwarp();
              tc_fence_after();
              const float f = grow ? ex2(m - mn) : 1.0f;
              l *= f;
#pragma unroll 1
              for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tO + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st_x32(tO + c, o);
              }
            }
            m = mn;
          }
          const float mu = m == -INFINITY ? 0.0f : m;
          const uint64_t nm2 = pair(-mu, -mu);
          uint64_t sum[2] = {0, 0};
          uint32_t p[HK / 2];
#pragma unroll
          for (int i = 0; i < HK / 2; ++i) {
            const uint64_t e2 = fma2(pair(s[2 * i], s[2 * i + 1]), c22, nm2);
            float e0, e1;
            unpair(e2, e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            sum[i & 1] = add2(sum[i & 1], pair(e0, e1));
            // Rounded to bf16 for the second product only; the sum keeps the
            // unrounded weights.
            p[i] = pack_bf16(e0, e1);
          }
          tmem_st_x16(tS + half * (HK / 2), p);
          float l0, l1;
          unpair(add2(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p + 8 * x);
        }
        // Every S of the item is done: its Q may go.
        have = !pair_any(!(next_seg() && ok));
        fetch = have && g.take > 0 && t < tiles(g);
        if (fetch) {
          q_start();
          q_done();
        }
        const uint32_t y = 2 * t + ((n - 1) & 1);
        ok = attn_wait(bar_o + 8 * y, ((n - 1) >> 1) & 1, status, kDevTimeoutAcc, abort) && ok;
        __syncwarp();
        tc_fence_after();
        l += pair_other(l);
      } else {
        have = !pair_any(!(next_seg() && ok));
        fetch = have && g.take > 0 && t < tiles(g);
        if (fetch) {
          q_start();
          q_done();
        }
      }
      if (!mine) continue;

      // ---- epilogue: straight from TMEM (shared memory is busy with the other
      // tile's MMAs), 16 rows at a time in the shape where 4
      // lanes hold 8 columns of a row side by side.  The loops stay rolled: this
      // code runs once per item and would come from L2 line by line.
      AttnFinish f = {};
      if (in) {
        if (slot < 0) {
          f = attn_finish(a, ar, m, l);
          if (half == 0) attn_store_lse(a, f);
        } else {
          if (half == 0) a.part_ml[(int64_t)slot * R + my] = make_float2(m, l);
          f.so = 1.0f;
        }
      }
      // MODE 0: fp32 rows (a part, or the prefix pass); 1: bf16 rows; 2: bf16
      // rows with a gate or the prefix's part joined.  A loop of its own each,
      // so that it runs without branches.
      auto store_rows = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
#pragma unroll 1
        for (int h = 0; h < 32; h += 16) {
          float so[2], sp[2];
          char *dst[2];  // this lane's first column of its two rows
          const char *gate[2], *prev[2];
          bool on[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int src = h + 8 * i + (lane >> 2);
            const int tok = __shfl_sync(0xffffffffu, ar.token, src), head = __shfl_sync(0xffffffffu, ar.head, src);
            const int64_t id = ((int64_t)tok * a.Hq + head) * DP + 2 * (lane & 3);
            on[i] = __shfl_sync(0xffffffffu, (int)in, src);
            so[i] = __shfl_sync(0xffffffffu, f.so, src);
            if constexpr (MODE == 0) {
              const int64_t pid = ((int64_t)slot * R + t * 128 + wq * 32 + src) * DP + 2 * (lane & 3);
              dst[i] = reinterpret_cast<char *>(slot >= 0 ? a.part_o + pid : a.prev_o + id);
            } else {
              dst[i] = reinterpret_cast<char *>(a.out + tok * a.o_ts + head * a.o_hs + 2 * (lane & 3));
            }
            if constexpr (MODE == 2) {
              sp[i] = __shfl_sync(0xffffffffu, f.sp, src);
              prev[i] = reinterpret_cast<const char *>(a.prev_o + id);
              gate[i] = reinterpret_cast<const char *>(a.gate + tok * a.g_ts + head * a.g_hs + 2 * (lane & 3));
            }
          }
          // This warp's half of the columns, 32 a step; 64 where there are registers
          // for the gate's and the prefix's loads of as many.
          constexpr int W = MODE == 2 && QT == 1 ? 64 : 32;
          const int cols = min(MODE == 0 ? DP : a.D, (half + 1) * (DP / 2));
#pragma unroll 1
          for (int c0 = half * (DP / 2); c0 < cols; c0 += W) {
            // Per row i: columns c0 + 8 k + 2 (lane % 4) + {0, 1}.
            uint32_t o[W / 32][16] = {}, w[2][W / 8] = {};
            float2 p[2][W / 8] = {};
            if (take > 0)
#pragma unroll
              for (int x = 0; x < W / 32; ++x) tmem_ld_16x256_x4(tO + ((uint32_t)h << 16) + c0 + 32 * x, o[x]);
            if constexpr (MODE == 2) {
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < W / 8; ++k) {
                  if (a.gate && on[i] && c0 + 8 * k < cols)
                    w[i][k] = *reinterpret_cast<const uint32_t *>(gate[i] + 2 * (c0 + 8 * k));
                  if (a.prev_o && sp[i] != 0.0f) p[i][k] = *reinterpret_cast<const float2 *>(prev[i] + 4 * (c0 + 8 * k));
                }
            }
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int k = 0; k < W / 8; ++k) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float v = __uint_as_float(o[k / 4][4 * (k % 4) + 2 * i + e]);
                  x[e] = so[i] == 0.0f ? 0.0f : v * so[i];
                  if constexpr (MODE == 2) {
                    x[e] = fmaf(e ? p[i][k].y : p[i][k].x, sp[i], x[e]);
                    const float g = sigmoidf(__uint_as_float(e ? w[i][k] & 0xffff0000u : w[i][k] << 16));
                    x[e] *= a.gate ? g : 1.0f;
                  }
                }
                if constexpr (MODE == 0) {
                  if (on[i]) *reinterpret_cast<float2 *>(dst[i] + 4 * (c0 + 8 * k)) = make_float2(x[0], x[1]);
                } else {
                  if (on[i] && c0 + 8 * k < cols)
                    *reinterpret_cast<uint32_t *>(dst[i] + 2 * (c0 + 8 * k)) = pack_bf16(x[0], x[1]);
                }
              }
          }
        }
      };
      if (slot >= 0 || a.prefix_pass) store_rows(std::integral_constant<int, 0>());
      else if (!a.gate && !a.prev_o) store_rows(std::integral_constant<int, 1>());
      else store_rows(std::integral_constant<int, 2>());
      tc_fence_before();
    }
  } else {
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int role = warp - C::kSoftWarps;
    if (role == 0 || (role == 3 && QT == 2)) {
      // ---------------- MMA issue, a warp per query tile ----------------
      const int t = role == 0 ? 0 : 1;
      constexpr uint32_t idS = idesc_bf16_f32(128, KT);
      constexpr uint32_t idO = idesc_bf16_f32(128, DP) | kTransposeB;
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), sb = __shfl_sync(0xffffffffu, sbase, 0);
      const uint32_t box = min(a.page_size, KT), b1 = box == 16 ? DP * 2 : 128, b2 = box == KT ? 256 : DP * 4;
      const uint32_t qd = desc_lo(sb + t * C::kQ, 16), kd = desc_lo(sb + C::offKV, 16),
                     vd = desc_lo(sb + C::offKV, box * 128);
      bool ok = true;
      // The slot of the next key tile's K (its V is in the slot after) and of
      // the pending tile's V, with the parities of their rounds.
      uint32_t slot = 0, round = 0, vslot = 0, vround = 0;
      uint32_t ns = 0, np = 0, nq = 0;  // S issued, P V issued, queries awaited
      bool pend = false, pfirst = false, puse = false, use = false, more = true;
      int u = 0, take = 0;  // pfirst, puse: of the pending P V
      auto wait = [&](uint32_t bar, uint32_t ph, int code) {
        ok = ok && __all_sync(0xffffffffu, attn_wait(bar, ph, status, code, abort));
      };
      auto pv = [&]() {
        wait(full + 8 * vslot, vround & 1, kDevTimeoutFull);
        if (puse) {
          const uint32_t x = 2 * t + (np & 1);
          wait(bar_p + 8 * x, (np >> 1) & 1, kDevTimeoutDec);
          ++np;
          if (ok) {
            tc_fence_after();
            mma_ts4(tm + C::colO + t * DP, tm + x * KT, vd + vslot * (C::kTile >> 4), idO, !pfirst, b1, b2);
            commit_to(bar_o + 8 * x);
          }
        }
        commit_to(empty + 8 * vslot);
        pend = false;
      };
      while (ok) {
        if (u == take) {  // the next item
          if (!next_seg()) more = false;
          u = 0;
          take = __shfl_sync(0xffffffffu, g.take, 0);
          use = t < __shfl_sync(0xffffffffu, tiles(g), 0);
          // An item's last P V comes before the next item's S, which may wait
          // for its queries.
          if (pend) pv();
          if (!more) break;
          if (take == 0) continue;
        }
        wait(full + 8 * slot, round & 1, kDevTimeoutFull);
        if (use) {  // S; within an item it goes before the P V of the tile before
          if (u == 0) wait(bar_q + 8 * t, nq++ & 1, kDevTimeoutDec);
          if (ok) {
            tc_fence_after();
            const uint32_t x = 2 * t + (ns++ & 1), k0 = kd + slot * (C::kTile >> 4);
#pragma unroll
            for (int hf = 0; hf < DP / 64; ++hf)
              mma_ss4(tm + x * KT, qd + hf * (128 * 128 >> 4), k0 + hf * (KT * 128 >> 4), idS, hf != 0);
            commit_to(bar_s + 8 * x);
          }
        }
        commit_to(empty + 8 * slot);
        if (pend && ok) pv();
        vslot = slot + 1 == kSlots ? 0 : slot + 1;
        vround = slot + 1 == kSlots ? round + 1 : round;
        slot = vslot + 1 == kSlots ? 0 : vslot + 1;
        round = vslot + 1 == kSlots ? vround + 1 : vround;
        pfirst = u == 0;
        puse = use;
        pend = true;
        ++u;
      }
      // TMEM is given back only when every MMA has finished.
      commit_to(bar_end);
      volatile int no_abort = 0;
      attn_wait(bar_end, 0, status, kDevTimeoutAcc, &no_abort);
      __syncwarp();
    } else if (role == 1) {
      // ---------------- TMA producer ----------------
      const int box = a.page_size < KT ? a.page_size : KT;
      const int per = KT / box;
      // This lane's box of a tile and its block of columns (wide: all of them).
      const int bi = lane % per, bx = lane / per;
      const uint64_t policy = l2_evict_normal_policy();
      uint32_t at = 0;
      bool ok = true;
      while (ok && next_seg()) {
        const int *pages = a.page_table + (a.prefix_pass ? 0 : (int64_t)g.b * a.pt_stride);
        const int take = __shfl_sync(0xffffffffu, g.take, 0), h = __shfl_sync(0xffffffffu, g.h, 0);
        const int lo = __shfl_sync(0xffffffffu, g.it.lo, 0), hi = __shfl_sync(0xffffffffu, g.it.hi, 0);
        int j0 = __shfl_sync(0xffffffffu, (g.it.u0 + g.off) * KT, 0);
        int ids = 0, ids_at = -64;
        for (int u = 0; u < take && ok; ++u, j0 += KT) {
          const int p0 = j0 >> a.page_shift, p1 = (j0 + KT - 1) >> a.page_shift;
          if (p1 >= ids_at + 32) {  // the next 32 page ids, one per lane
            ids_at = p0;
            ids = pages[min(p0 + lane, (hi - 1) >> a.page_shift)];
          }
          const bool ragged = j0 < lo || j0 + KT > hi;
          const int tok = j0 + bi * box;
          const bool seen = tok < hi && tok + box > lo;  // holds a key that some row sees
          const int page = __shfl_sync(0xffffffffu, ids, ((tok >> a.page_shift) - ids_at) & 31);
          const int row = tok & (a.page_size - 1);
          for (int kv = 0; kv < 2; ++kv, ++at) {
            const bool all = kv ? a.wide_v : a.wide;
            const bool mine = seen && bx < (all ? 1 : DP / 64);
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * box * (all ? DP * 2 : 128);
            const uint32_t slot = at % kSlots, round = at / kSlots;
            if (round > 0 && !__all_sync(0xffffffffu, attn_wait(empty + 8 * slot, (round - 1) & 1, status,
                                                                kDevTimeoutEmpty, abort))) {
              ok = false;
              break;
            }
            const uint32_t bar = (kv && ragged ? edge : full) + 8 * slot;
            if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (mine)
              attn_load_box(sbase + C::offKV + slot * C::kTile + (kv ? bi * (DP / 64) + bx : bx * per + bi) * box * 128, kv ? &tmV : &tmK,
                            64 * bx, row, h, page, bar, policy);
          }
        }
      }
      // Drain: the block never exits with a copy still writing its memory.
      for (uint32_t q = at > kSlots ? at - kSlots : 0; q < at; ++q) {
        volatile int no_abort = 0;
        attn_wait(full + 8 * (q % kSlots), (q / kSlots) & 1, status, kDevTimeoutFull, &no_abort);
      }
    } else if (role == 2) {
      // ---------------- values that no row sees ----------------
      // Rows of a value tile before the first or from the last key on (never
      // loaded, or the rest of a page) are zeroed: their weights are zero,
      // but what lies there may not be finite.
      // This warp also lists the block's items, three ahead of its own.
      uint32_t at = 0, phase = 0, listed = 0;
      bool ok = true, more = true;
      while (ok) {
        if (lane == 0) {
          for (; more && listed < nseg + kSegs - 1; ++listed) {
            const uint32_t i = listed % kSegs;
            if (listed >= kSegs &&
                !attn_wait(seg_empty + 8 * i, (listed / kSegs - 1) & 1, status, kDevTimeoutEmpty, abort))
              break;
            more = attn_segment<R, KT, E>(a, cur, g);
            if (!more) g.take = -1;
            segs[i] = g;
            mbar_arrive(seg_full + 8 * i);
          }
        }
        __syncwarp();
        if (!next_seg()) break;
        for (int u = 0; u < g.take; ++u, at += 2) {
          const int j0 = (g.it.u0 + g.off + u) * KT;
          if (j0 >= g.it.lo && j0 + KT <= g.it.hi) continue;
          const uint32_t slot = (at + 1) % kSlots;
          if (!__all_sync(0xffffffffu, attn_wait(edge + 8 * slot, (phase >> slot) & 1, status,
                                                 kDevTimeoutFull, abort))) {
            ok = false;
            break;
          }
          phase ^= 1u << slot;
          uint8_t *V = smem + C::offKV + slot * C::kTile;
          const int box = a.page_size < KT ? a.page_size : KT;
          for (int x = lane; x < KT * (DP / 8); x += 32) {
            const int r = x / (DP / 8), c = x % (DP / 8), j = j0 + r, in = r & (box - 1);
            if (j < g.it.lo || j >= g.it.hi)
              *reinterpret_cast<uint4 *>(V + ((r - in) * (DP / 64) + (c >> 3) * box + in) * 128 +
                                         (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full + 8 * slot);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kSoftWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, C::cols);
  }
}

template <int DP>
cudaError_t launch_tc(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int grid,
                      cudaStream_t st) {
  using C = TcCfg<DP>;
  const bool mod = a.softcap > 0.0f || a.slopes;
  auto k = mod ? attn_tc_kernel<DP, true> : attn_tc_kernel<DP, false>;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t e = attn_allow_smem(reinterpret_cast<const void *>(k), C::bytes, allowed[mod]);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, k, tk, tv, a)) != cudaSuccess) return e;
  constexpr int RPB = 8;
  const int rows = a.max_rows < C::R ? a.max_rows : C::R;
  cfg.gridDim = dim3((unsigned)grid, (unsigned)((rows + RPB - 1) / RPB), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attn_join_kernel<C::R, DP, 1, RPB>, a);
}

}  // namespace

cudaError_t launch_attn_tc(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int grid,
                           cudaStream_t st) {
  if (a.D <= 64) return launch_tc<64>(tk, tv, a, grid, st);
  if (a.D <= 128) return launch_tc<128>(tk, tv, a, grid, st);
  return launch_tc<256>(tk, tv, a, grid, st);
}

int read_attn_tc_device_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_tc_status, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_attn_tc_status, &zero, sizeof(int));
  return v;
}

}  // namespace nvfp4
