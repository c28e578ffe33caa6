// attention_tc.cu -- attention of many query rows per key/value head (prompts,
// a shared prefix) over the paged cache, on the 5th-generation tensor cores.
//
// An item is QT tiles of 128 query rows (attention.cuh: the heads of a group
// share their keys, so 8 heads make a tile of 16 tokens).  Per key tile j and
// query tile t: S = Q K_j^T into TMEM, a softmax thread per row, P as bf16
// back into TMEM over S, O += P V_j with P as the TMEM operand and V in its
// natural token-major layout (MN-major operand).  O stays in TMEM for all of
// an item.  Up to head size 128 QT = 2 and the two tiles alternate: while one
// is in its softmax the other has the tensor cores.  Above, O takes half of
// TMEM: QT = 1 and two S buffers, the next S running under the softmax.
//   warps 0-3 (and 4-7, QT = 2)  softmax of tile 0 (1), Q into shared memory,
//                                the rare rescaling of O, the epilogue;
//   then one warp each           MMA issue (one thread), TMA producer, zeroing
//                                of values that no row sees, and the block's
//                                list of items.
// O is rescaled only when a row's maximum has grown by more than 2^8 since
// the last time (weights then stay below 2^8, exact in the sums' fp32); the
// reference is the same for sum and product, so the result is not changed.
// Bound by the tensor cores and, nearly as much, by the exponentials: 2 x 128
// x 128 of them per 2048 tensor cycles are 2048 cycles of the MUFU.
#include <cuda_bf16.h>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention.cuh"
#include "attention_launch.h"
#include "kernels.h"
#include "tc_common.cuh"

namespace nvfp4 {

static __device__ int g_attn_tc_status;

namespace {

constexpr int kItemCost = 1;  // of an item's beginning and end, in key tiles
constexpr int kSegs = 4;      // items that the scheduling warp may be ahead

template <int DP>
struct TcCfg {
  static constexpr int QT = DP <= 128 ? 2 : 1;
  static constexpr int R = 128 * QT;
  static constexpr int KT = DP <= 128 ? 128 : 64;   // keys per tile
  static constexpr int kTile = KT * DP * 2;         // bytes of a key or value tile
  static constexpr int kQ = 128 * DP * 2;           // bytes of a query tile
  static constexpr int kSlots = DP == 64 ? 8 : 4;
  static constexpr int kSoftWarps = 4 * QT;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;
  static constexpr int offKV = QT * kQ;
  static constexpr int offStage = offKV + kSlots * kTile;  // 2 KB per softmax warp
  static constexpr int bytes = offStage + kSoftWarps * 2048 + 1024;
  // TMEM columns: S tiles (tile t, or buffer t when QT = 1), then O.
  static constexpr int colO = 2 * KT;
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
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem].
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Values [token][d], 64 columns of 128 swizzled bytes per token, as the
// MN-major B operand: 64-column blocks `block` bytes apart (leading offset),
// groups of 8 tokens 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr, uint32_t block) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
constexpr uint32_t kTransposeB = 1u << 16;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int h, int row,
                                            int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(row), "r"(page), "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <int DP, bool MOD>
__global__ void __launch_bounds__(TcCfg<DP>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ AttnArgs a) {
  using C = TcCfg<DP>;
  constexpr int QT = C::QT, R = C::R, KT = C::KT, kSlots = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  __shared__ AttnPlanSmem plan;
  __shared__ uint64_t bars[3 * kSlots + 9 + 2 * kSegs];
  __shared__ AttnSegment segs[kSegs];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full = smem_u32(bars);
  const uint32_t empty = full + 8 * kSlots;   // the slot's MMAs are done
  const uint32_t edge = empty + 8 * kSlots;   // a value tile landed that needs zeroing
  const uint32_t bar_q = edge + 8 * kSlots;   // [2] queries of tile t in shared memory
  const uint32_t bar_s = bar_q + 16;          // [2] S ready
  const uint32_t bar_p = bar_s + 16;          // [2] P written (and O rescaled)
  const uint32_t bar_o = bar_p + 16;          // [2] P V done (tile t; QT = 1: even and odd products)
  const uint32_t bar_end = bar_o + 16;
  const uint32_t seg_full = bar_end + 8;      // [kSegs] the block's next items
  const uint32_t seg_empty = seg_full + 8 * kSegs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
      mbar_init(edge + 8 * i, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_q + 8 * t, 4);
      mbar_init(bar_s + 8 * t, 1);
      mbar_init(bar_p + 8 * t, 4);
      mbar_init(bar_o + 8 * t, 1);
    }
    mbar_init(bar_end, 1);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(seg_full + 8 * i, 1);
      mbar_init(seg_empty + 8 * i, C::kSoftWarps + 3);
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
  AttnCursor cur = attn_plan<R, KT, kItemCost>(a, 2 + kItemCost, &plan);  // ends with __syncthreads
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t tmem = tmem_slot;
  if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, -1);
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
    if constexpr (QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, wq = warp & 3;            // tile, lane quarter
    const int my = t * 128 + wq * 32 + lane;           // row within the item
    const uint32_t lanes = static_cast<uint32_t>(32 * wq) << 16;
    const uint32_t tO = tmem + lanes + C::colO + (QT == 2 ? t * DP : 0);
    uint8_t *Q = smem + t * C::kQ;
    const float sl2 = a.scale * kLog2e;

    // This warp's 32 rows of Q, 16-byte chunks swizzled as the MMA reads them;
    // rows and columns beyond the item's or the head's are zeros.
    auto load_q = [&]() {
      const AttnSegment &x = g;
      const int row = x.rb * R + my;
      const __nv_bfloat16 *src = nullptr;
      if (row < x.s.ql * a.G) {
        const int i = row / a.G;
        src = a.q + (int64_t)(x.s.tok0 + i) * a.q_ts + (int64_t)(x.h * a.G + row - i * a.G) * a.q_hs;
      }
      constexpr int CH = DP / 8, RPI = 32 / CH;  // chunks per row, rows per warp step
      const int c = lane % CH;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += RPI) {
        const int r = r0 + lane / CH;
        const uint64_t p = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), r);
        const int rr = wq * 32 + r;
        const bool on = p != 0 && 8 * c < a.D;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         smem_u32(Q + (c >> 3) * (128 * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4))),
                     "l"(on ? p + 16 * c : reinterpret_cast<uint64_t>(a.q)), "r"(on ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 8 * t);
    };

    // Product i of this query tile is in.  With QT = 1 the S that is ready
    // may be ahead of the last two products, so these alternate between two
    // barriers: each then has at most one phase outstanding.
    auto o_wait = [&](uint32_t i) {
      return QT == 2 ? attn_wait(bar_o + 8 * t, i & 1, status, kDevTimeoutAcc, abort)
                     : attn_wait(bar_o + 8 * (i & 1), (i >> 1) & 1, status, kDevTimeoutAcc, abort);
    };
    uint32_t n = 0;  // key tiles of this query tile so far
    bool have = next_seg(), ok = true;
    if (have && g.take > 0 && t < tiles(g)) load_q();
    while (have && ok) {
      const bool mine = t < tiles(g);
      const int row = g.rb * R + my;
      const bool in = row < g.s.ql * a.G;
      AttnRow ar = {};
      float m = -INFINITY, l = 0.0f;
      if (mine) {
        ar = attn_row(a, g.s, g.h, in ? row : 0);
        if (!in) ar.lo = ar.hi = 0;
        const float slope = MOD && a.slopes ? a.slopes[ar.head] * kLog2e : 0.0f;
        const int pos = ar.pos - (a.prefix_pass ? 0 : a.prefix_len);
        for (int u = 0; u < g.take; ++u, ++n) {
          const int j0 = (g.it.u0 + g.off + u) * KT;
          const int b = QT == 2 ? t : (n & 1);
          const uint32_t ph = QT == 2 ? n & 1 : (n >> 1) & 1;
          const uint32_t tS = tmem + lanes + b * KT;
          if (!__all_sync(0xffffffffu, attn_wait(bar_s + 8 * b, ph, status, kDevTimeoutAcc, abort))) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t raw[KT / 32][32];
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) tmem_ld_32x32b_x32(tS + 32 * c, raw[c]);
          tmem_ld_wait();
          float s[KT];
#pragma unroll
          for (int c = 0; c < KT; ++c) s[c] = __uint_as_float(raw[c / 32][c % 32]);
          if constexpr (MOD) {
#pragma unroll
            for (int c = 0; c < KT; ++c) {
              float v = s[c] * a.scale;
              if (a.softcap > 0.0f)  // cap tanh(v / cap)
                v = a.softcap - __fdividef(2.0f * a.softcap, 1.0f + ex2(v * (2.0f * kLog2e / a.softcap)));
              s[c] = fmaf(v, kLog2e, -slope * fabsf((float)(pos - j0 - c)));
            }
          }
          const float c2 = MOD ? 1.0f : sl2;
          if (__any_sync(0xffffffffu, j0 < ar.lo || j0 + KT > ar.hi)) {
            const int lo = ar.lo - j0, hi = ar.hi - j0;
#pragma unroll
            for (int c = 0; c < KT; ++c) s[c] = c >= lo && c < hi ? s[c] : -INFINITY;
          }
          float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int c = 4; c < KT; c += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], s[c + i]);
          const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c2;
          const bool grow = mx > m + 8.0f;
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? mx : m;
            if (u > 0) {  // O of the tiles before, once they are all in
              if (!__all_sync(0xffffffffu, o_wait(n - 1))) {
                ok = false;
                break;
              }
              tc_fence_after();
              const float f = grow ? ex2(m - mn) : 1.0f;
              l *= f;
#pragma unroll 1
              for (int c = 0; c < DP; c += 32) {
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
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < KT; c += 64) {
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = ex2(fmaf(s[c + 2 * i], c2, -mu)), y = ex2(fmaf(s[c + 2 * i + 1], c2, -mu));
              sum[(2 * i) & 3] += x;
              sum[(2 * i + 1) & 3] += y;
              // Rounded to bf16 for the second product only; the sum keeps
              // the unrounded weights.
              p[i] = pack_bf16(x, y);
            }
            tmem_st_x32(tS + c / 2, p);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p + 8 * b);
        }
      }
      if (!ok) break;
      // The next item's queries first (this item's S are all done), so that
      // its first S runs under this epilogue.
      const int e_take = g.take, e_slot = g.slot, e_rb = g.rb;
      if (g.last_part >= 0 && threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(g.b, g.h, g.rb, g.last_part);
      const int left = min(g.s.ql * a.G - e_rb * R - t * 128 - wq * 32, 32);  // this warp's rows in use
      have = next_seg();
      if (have && g.take > 0 && t < tiles(g)) load_q();
      if (!mine) continue;
      if (e_take > 0) {
        if (!__all_sync(0xffffffffu, o_wait(n - 1))) break;
        tc_fence_after();
      }
      // O by way of shared memory, 16 columns at a time, so that 4 lanes
      // store 16 columns of a row side by side.
      AttnFinish f = {};
      if (in && e_slot < 0) {
        f = attn_finish(a, ar, m, l);
        attn_store_lse(a, f);
      }
      if (in && e_slot >= 0) a.part_ml[(int64_t)e_slot * R + my] = make_float2(m, l);
      // This lane's 4 rows of a step, at its 4 columns.
      const int64_t id = in ? (int64_t)ar.token * a.Hq + ar.head : 0;
      const float so = e_slot < 0 ? f.so : 1.0f;
      int64_t at[4], gat[4], pat[4];
      float sp[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int src = 8 * i + (lane >> 2);
        const int tok = __shfl_sync(0xffffffffu, ar.token, src), head = __shfl_sync(0xffffffffu, ar.head, src);
        pat[i] = __shfl_sync(0xffffffffu, id, src) * DP;
        if (e_slot >= 0) at[i] = ((int64_t)e_slot * R + t * 128 + wq * 32 + src) * DP;
        else if (a.prefix_pass) at[i] = pat[i];
        else at[i] = tok * a.o_ts + head * a.o_hs;
        gat[i] = tok * a.g_ts + head * a.g_hs;
        sp[i] = __shfl_sync(0xffffffffu, f.sp, src);
      }
      const bool to_f32 = e_slot >= 0 || a.prefix_pass, joins = !to_f32 && a.prev_o, gates = !to_f32 && a.gate;
      float *f32 = e_slot >= 0 ? a.part_o : a.prev_o;
      const uint32_t stage = sbase + C::offStage + warp * 2048;
      const uint32_t st_w = stage + lane * 64, x_w = (lane >> 1) & 3;
      // The gates come a step ahead of their use.
      auto load_gates = [&](uint2 (&v)[4], int d) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (gates && 8 * i + (lane >> 2) < left && d < a.D)
            v[i] = *reinterpret_cast<const uint2 *>(a.gate + gat[i] + d);
      };
      uint2 gv[4] = {}, gn[4] = {};
      load_gates(gn, 4 * (lane & 3));
#pragma unroll 1
      for (int c = 0; c < DP; c += 16) {
        const int d = c + 4 * (lane & 3);
        uint32_t o[16] = {};
        if (e_take > 0) tmem_ld_x16(tO + c, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) gv[i] = gn[i];
        if (c + 16 < DP) load_gates(gn, d + 16);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = so == 0.0f ? 0.0f : __uint_as_float(o[4 * i + x]) * so;
          asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(st_w + ((i ^ x_w) << 4)), "f"(v[0]),
                       "f"(v[1]), "f"(v[2]), "f"(v[3])
                       : "memory");
        }
        __syncwarp();
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2);
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                       : "=f"(x[i].x), "=f"(x[i].y), "=f"(x[i].z), "=f"(x[i].w)
                       : "r"(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4))
                       : "memory");
        }
        __syncwarp();
        if (d >= a.D) continue;
        if (to_f32) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (8 * i + (lane >> 2) < left) *reinterpret_cast<float4 *>(f32 + at[i] + d) = x[i];
          continue;
        }
        if (joins) {
          float4 p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = make_float4(0, 0, 0, 0);
            if (sp[i] != 0.0f) p[i] = *reinterpret_cast<const float4 *>(a.prev_o + pat[i] + d);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i].x = fmaf(p[i].x, sp[i], x[i].x);
            x[i].y = fmaf(p[i].y, sp[i], x[i].y);
            x[i].z = fmaf(p[i].z, sp[i], x[i].z);
            x[i].w = fmaf(p[i].w, sp[i], x[i].w);
          }
        }
        if (gates) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i].x *= sigmoidf(__uint_as_float(gv[i].x << 16));
            x[i].y *= sigmoidf(__uint_as_float(gv[i].x & 0xffff0000u));
            x[i].z *= sigmoidf(__uint_as_float(gv[i].y << 16));
            x[i].w *= sigmoidf(__uint_as_float(gv[i].y & 0xffff0000u));
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (8 * i + (lane >> 2) < left)
            *reinterpret_cast<uint2 *>(a.out + at[i] + d) =
                make_uint2(pack_bf16(x[i].x, x[i].y), pack_bf16(x[i].z, x[i].w));
      }
      tc_fence_before();
    }
  } else {
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int role = warp - C::kSoftWarps;
    if (role == 0) {
      // ---------------- MMA issue ----------------
      if (lane == 0) {
        constexpr uint32_t idS = idesc_bf16_f32(128, KT);
        constexpr uint32_t idO = idesc_bf16_f32(128, DP) | kTransposeB;
        bool ok = true;
        uint32_t tile = 0;       // key tiles so far: K in slot 2 tile, V in 2 tile + 1
        uint32_t ns[2] = {0, 0}; // S issued per query tile
        uint32_t nq[2] = {0, 0}; // queries awaited per query tile
        bool pend = false, pfirst = false, more = true;
        int pnt = 0, u = 0, nt = 0;  // pnt, pfirst: of the pending P V
        g.take = 0;
        auto wait = [&](uint32_t bar, uint32_t ph, int code) {
          ok = ok && attn_wait(bar, ph, status, code, abort);
        };
        while (ok && (more || pend)) {
          // The next key tile, if any; P V of the tile before it is pending.
          if (more && u == g.take) {
            do {
              const uint32_t i = nseg % kSegs;
              wait(seg_full + 8 * i, (nseg / kSegs) & 1, kDevTimeoutDec);
              if (!ok) break;
              g = segs[i];
              mbar_arrive(seg_empty + 8 * i);
              ++nseg;
            } while (g.take == 0);
            if (!ok) break;
            more = g.take > 0;
            u = 0;
            nt = tiles(g);
          }
          // In which order: bits 0, 1 the query tile, bit 2 a P V, bit 3 none.
          // Within an item QT = 2 alternates P V and S of the two tiles and
          // QT = 1 keeps one S ahead; an item's last P V come before the next
          // item's S, which may wait for its queries.
          uint32_t ops;
          const bool inner = more && pend && u > 0;
          if (QT == 2) ops = inner ? 0x1504 : 0x1054;
          else ops = inner ? 0x8840 : 0x8804;
          if (!pend || pnt < 2) ops |= QT == 2 ? (inner ? 0x0800 : 0x0080) : 0;
          if (!pend) ops |= QT == 2 ? 0x0008 : (inner ? 0x0080 : 0x0008);
          if (!more) ops |= QT == 2 ? 0x8800 : 0x0080;
          if (more && nt < 2 && QT == 2) ops |= 0x8000;
          bool v_in = false, k_in = false;
#pragma unroll 1
          for (; ops != 0x8888 && ok; ops = (ops >> 4) | 0x8000) {
            const int op = ops & 15, t = op & 3;
            if (op & 8) continue;
            if (op & 4) {
              if (!v_in) wait(full + 8 * ((2 * tile - 1) % kSlots), ((2 * tile - 1) / kSlots) & 1, kDevTimeoutFull);
              v_in = true;
              const uint32_t np = QT == 2 ? ns[t] - 1 : tile - 1;  // this P V's count
              const int b = QT == 2 ? t : (np & 1);
              wait(bar_p + 8 * b, (QT == 2 ? np : np >> 1) & 1, kDevTimeoutDec);
              if (!ok) break;
              tc_fence_after();
              const uint64_t v0 =
                  sw128_mnmajor_desc(sbase + C::offKV + ((2 * tile - 1) % kSlots) * C::kTile, KT * 128);
              const uint32_t d = tmem + C::colO + (QT == 2 ? t * DP : 0), p = tmem + b * KT;
#pragma unroll
              for (int k = 0; k < KT / 16; ++k)
                tc_mma_f16_ts(d, p + 8 * k, v0 + k * (2048 >> 4), idO, !(pfirst && k == 0));
              tc_commit(bar_o + 8 * (QT == 2 ? t : (np & 1)));
            } else {
              if (!k_in) wait(full + 8 * ((2 * tile) % kSlots), ((2 * tile) / kSlots) & 1, kDevTimeoutFull);
              k_in = true;
              if (u == 0) wait(bar_q + 8 * t, nq[t]++ & 1, kDevTimeoutDec);
              if (!ok) break;
              tc_fence_after();
              const int b = QT == 2 ? t : (ns[0] & 1);
              const uint64_t k0 = sw128_kmajor_desc(sbase + C::offKV + ((2 * tile) % kSlots) * C::kTile);
              const uint64_t q0 = sw128_kmajor_desc(sbase + t * C::kQ);
#pragma unroll
              for (int k = 0; k < DP / 16; ++k)
                tc_mma_f16(tmem + b * KT, q0 + (((k >> 2) * (128 * 128) + 32 * (k & 3)) >> 4),
                           k0 + (((k >> 2) * (KT * 128) + 32 * (k & 3)) >> 4), idS, k != 0);
              tc_commit(bar_s + 8 * b);
              ++ns[t];
            }
          }
          if (pend) tc_commit(empty + 8 * ((2 * tile - 1) % kSlots));
          if (more) {
            tc_commit(empty + 8 * ((2 * tile) % kSlots));
            pfirst = u == 0;
            pnt = nt;
            ++u;
            ++tile;
          }
          pend = more;
        }
        // TMEM is given back only when every MMA has finished.
        tc_commit(bar_end);
        volatile int no_abort = 0;
        attn_wait(bar_end, 0, status, kDevTimeoutAcc, &no_abort);
      }
      __syncwarp();
    } else if (role == 1) {
      // ---------------- TMA producer ----------------
      const int box = a.page_size < KT ? a.page_size : KT;
      const int per = KT / box;
      constexpr int halves = DP / 64;
      uint32_t at = 0;
      bool ok = true;
      while (ok && next_seg()) {
        const int *pages = a.page_table + (a.prefix_pass ? 0 : (int64_t)g.b * a.pt_stride);
        int ids = 0, ids_at = -64;
        for (int u = 0; u < g.take && ok; ++u) {
          const int j0 = (g.it.u0 + g.off + u) * KT;
          const int i = lane % per, hf = lane / per;
          const int tok = j0 + i * box;
          const bool mine = hf < halves && tok < g.it.hi && tok + box > g.it.lo;
          const int p0 = j0 >> a.page_shift, p1 = (j0 + KT - 1) >> a.page_shift;
          if (p1 >= ids_at + 32 || p0 < ids_at) {
            ids_at = p0;
            ids = pages[min(p0 + lane, (g.it.hi - 1) >> a.page_shift)];
          }
          const int page = __shfl_sync(0xffffffffu, ids, ((tok >> a.page_shift) - ids_at) & 31);
          const int row = tok & (a.page_size - 1);
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * box * 128;
          const bool ragged = j0 < g.it.lo || j0 + KT > g.it.hi;
          for (int kv = 0; kv < 2; ++kv, ++at) {
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
              tma_load_4d(sbase + C::offKV + slot * C::kTile + hf * (KT * 128) + i * box * 128,
                          kv ? &tmV : &tmK, 64 * hf, g.h, row, page, bar);
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
      uint32_t at = 0, phase = 0;
      bool ok = true;
      while (ok && next_seg()) {
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
          for (int x = lane; x < KT * (DP / 8); x += 32) {
            const int r = x / (DP / 8), c = x % (DP / 8), j = j0 + r;
            if (j < g.it.lo || j >= g.it.hi)
              *reinterpret_cast<uint4 *>(V + (c >> 3) * (KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full + 8 * slot);
        }
      }
    } else if (lane == 0) {
      // ---------------- the block's items, ahead of the other warps --------
      for (uint32_t n = 0;; ++n) {
        const uint32_t i = n % kSegs;
        if (n >= kSegs && !attn_wait(seg_empty + 8 * i, (n / kSegs - 1) & 1, status, kDevTimeoutEmpty, abort)) break;
        const bool more = attn_segment<R, KT, kItemCost>(a, cur, g);
        if (!more) g.take = -1;
        segs[i] = g;
        mbar_arrive(seg_full + 8 * i);
        if (!more) break;
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
  auto k = a.softcap > 0.0f || a.slopes ? attn_tc_kernel<DP, true> : attn_tc_kernel<DP, false>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::bytes);
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
  cfg.gridDim = dim3((unsigned)grid, C::R / 4, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attn_join_kernel<C::R, C::KT, DP>, a);
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
