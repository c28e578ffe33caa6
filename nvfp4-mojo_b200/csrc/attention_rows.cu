// attention_rows.cu -- attention of few query rows per key/value head (single
// tokens, a few tokens of speculative decoding) over the paged cache.
//
// Bound by HBM: every key and value is read once for the R = 16 rows (32 at head
// sizes up to 64) that share it, in one launch whose warps divide all sequences' keys evenly
// (attention.cuh), so a batch of ragged lengths keeps every SM streaming to
// the end.  Each of a block's eight warps works alone, without a barrier: it
// keeps key and value tiles of 32 tokens (16 above head size 128) in flight by TMA
// (a box per page, 128-byte swizzle), across the ends of its items, and turns
// each into S = Q K^T, its softmax state and O += P V on mma.sync from registers
// (16 rows would fill an eighth of a tcgen05 tile).  A cut item's parts go to
// the workspace as they are; there is nothing to join within a block.
//
// Measured with the join: 64 sequences of 200 to 12000 keys, 32 / 4 heads of 128,
// 131 us, 5.8 of the 6.6 TB/s that a copy reaches; 6 of 9000 to 60000 keys, 16 / 2
// heads of 256, with gate and log-sum-exp 77 us, 4.9 TB/s (12 items are cut into
// 1184 parts, whose join is 10 us of it).  One sequence of 650 keys takes 12.7 us:
// 2 us for the plan, 2 to the first tile, 3 for its three tiles, 1 for its end and
// 3 to 4 for the join, each the latency of a few dependent loads.
#include <cuda_bf16.h>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention.cuh"
#include "attention_launch.h"
#include "tc_common.cuh"

namespace nvfp4 {

static __device__ int g_attn_rows_status;
static_assert(kAttnRowsWorkers == 8, "warps per block below");

namespace {

constexpr int kWarps = 8;
// Of an item's beginning and end, in tiles.  (256 sequences of up to 400 keys:
// 41.5 us with 0, 40.6 with 1, 41.9 with 3.)
constexpr int kItemCost = 1;
constexpr int kSegs = 4;      // items that a warp's loads may be ahead

template <int MT, int DP>
struct RowsCfg {
  static constexpr int R = 16 * MT;
  static constexpr int KT = DP <= 128 ? 32 : 16;  // tokens per tile
  static constexpr int kTile = KT * DP * 2;       // bytes of a tile's keys, or values
  static constexpr int kRing = DP == 64 ? 6 : 3;  // tiles (keys or values) per warp
  static constexpr int bytes = kWarps * kRing * kTile + 1024;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// MOD: scores are capped or biased.
template <int MT, int DP, bool MOD>
__global__ void __launch_bounds__(kWarps * 32, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ AttnArgs a) {
  using C = RowsCfg<MT, DP>;
  constexpr int R = C::R, KT = C::KT, kRing = C::kRing, NT = KT / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  __shared__ AttnPlanSmem plan;
  __shared__ uint64_t bars[kWarps * kRing];
  __shared__ AttnSegment segs[kWarps][kSegs];
  __shared__ AttnCursor curs[kWarps];
  __shared__ int aborts[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full = smem_u32(bars + warp * kRing);
  uint8_t *ring = smem + warp * kRing * C::kTile;
  const uint32_t rbase = smem_u32(ring);

  asm volatile("griddepcontrol.launch_dependents;");
  if (lane == 0) {
    aborts[warp] = 0;
    for (int i = 0; i < kRing; ++i) mbar_init(full + 8 * i, 1);
    mbar_fence_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  {
    const AttnCursor c = attn_plan<R, KT, kItemCost, kWarps>(a, 1 + kItemCost, &plan, 0);
    if (lane == 0) {
      curs[warp] = c;
      a.meta[c.worker].last_part = -1;
    }
  }
  __syncwarp();
  volatile int *abort = &aborts[warp];
  int *status = &g_attn_rows_status;

  // Loads run up to kRing tiles (keys and values in turn) ahead of the
  // arithmetic.  The items lie in
  // shared memory; registers hold what every tile needs.
  int l_left = 0, l_j0 = 0, l_lo = 0, l_hi = 0, l_h = 0;  // the item being loaded
  const int *l_pages = nullptr;
  bool l_v = false;                                       // its next copy is of values
  int ids = 0, ids_at = -64;
  int take = 0, j0 = 0, it_lo = 0, it_hi = 0;             // the item being computed: tiles left
  uint32_t issued = 0, done = 0, pushed = 0, popped = 0;
  bool more = true, have = false;
  // A tile lies in shared memory box by box (a page's rows), a box as blocks
  // of 64 columns; 16 rows never cross a box.
  const int box = a.page_size < KT ? a.page_size : KT;
  const int per = KT / box, blocks = a.wide ? 1 : DP / 64;  // boxes per tile, copies per box
  const int bi = lane % per, bx = lane / per;               // this lane's copy
  const uint32_t cstride = box * 128;                     // from 64 columns to the next
  const uint32_t rstride = box == 16 ? 16 * DP * 2 : 16 * 128;  // from 16 rows to the next
  const uint64_t policy = l2_evict_first_policy();

  const int qr = lane >> 2, qc = lane & 3;
  const float sl2 = a.scale * kLog2e;
  uint32_t qf[MT][DP / 16][4];
  int lo[MT][2], hi[MT][2], pos[MT][2];
  float slope[MT][2], m[MT][2], l[MT][2], o[MT][DP / 8][4];

  while (true) {
    // ---- loads
#pragma unroll 1
    while (more && issued - done < kRing && (l_left > 0 || pushed - popped < kSegs)) {
      if (l_left == 0) {
        AttnCursor c = curs[warp];
        AttnSegment g;
        more = attn_segment<R, KT, kItemCost>(a, c, g);
        if (!more) break;
        __syncwarp();
        if (lane == 0) {
          curs[warp] = c;
          segs[warp][pushed % kSegs] = g;
        }
        __syncwarp();
        ++pushed;
        l_left = g.take;
        l_j0 = (g.it.u0 + g.off) * KT;
        l_lo = g.it.lo;
        l_hi = g.it.hi;
        l_h = g.h;
        l_pages = a.page_table + (a.prefix_pass ? 0 : (int64_t)g.b * a.pt_stride);
        ids_at = -64;
        continue;
      }
      const int p0 = l_j0 >> a.page_shift, p1 = (l_j0 + KT - 1) >> a.page_shift;
      if (p1 >= ids_at + 32) {  // the next 32 page ids, one per lane
        ids_at = p0;
        ids = l_pages[min(p0 + lane, (l_hi - 1) >> a.page_shift)];
      }
      const uint32_t st = issued % kRing;
      const int tok = l_j0 + bi * box;
      const bool mine = bx < blocks && tok < l_hi && tok + box > l_lo;  // holds a key that some row sees
      const int page = __shfl_sync(0xffffffffu, ids, ((tok >> a.page_shift) - ids_at) & 31);
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * box * (a.wide ? DP * 2 : 128);
      if (lane == 0) mbar_arrive_expect_tx(full + 8 * st, bytes);
      __syncwarp();
      if (mine)
        attn_load_box(rbase + st * C::kTile + bi * box * DP * 2 + bx * cstride, l_v ? &tmV : &tmK, 64 * bx,
                      tok & (a.page_size - 1), l_h, page, full + 8 * st, policy);
      ++issued;
      if (l_v) {
        l_j0 += KT;
        --l_left;
      }
      l_v = !l_v;
    }
    // ---- the next item
    if (!have) {
      if (popped == pushed) break;
      const AttnSegment &g = segs[warp][popped % kSegs];
      have = true;
      take = g.take;
      j0 = (g.it.u0 + g.off) * KT;
      it_lo = g.it.lo;
      it_hi = g.it.hi;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t *src[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = g.rb * R + mt * 16 + e * 8 + qr;
          const bool in = row < g.s.ql * a.G;
          const AttnRow r = attn_row(a, g.s, g.h, in ? row : 0);
          lo[mt][e] = in ? r.lo : 0;
          hi[mt][e] = in ? r.hi : 0;
          pos[mt][e] = r.pos - (a.prefix_pass ? 0 : a.prefix_len);
          slope[mt][e] = MOD && a.slopes ? a.slopes[r.head] * kLog2e : 0.0f;
          src[e] = in ? reinterpret_cast<const uint32_t *>(a.q + r.token * a.q_ts + r.head * a.q_hs) : nullptr;
          m[mt][e] = -INFINITY;
          l[mt][e] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int d = 16 * k + 8 * (x >> 1) + 2 * qc;
            qf[mt][k][x] = src[x & 1] && d < a.D ? src[x & 1][d >> 1] : 0u;
          }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[mt][n][x] = 0.0f;
      }
    }
    // ---- a tile
    if (take > 0) {
      const uint32_t st = done % kRing;
      if (!__all_sync(0xffffffffu, attn_wait(full + 8 * st, (done / kRing) & 1, status, kDevTimeoutFull, abort)))
        break;
      const uint32_t sv = (done + 1) % kRing, kb0 = rbase + st * C::kTile, vb0 = rbase + sv * C::kTile;
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][n][x] = 0.0f;
      {  // S = Q K^T: matrix lane / 8 holds tokens 8 (lane / 16), columns 8 ((lane / 8) & 1)
        const int t = (lane & 7) + 8 * (lane >> 4), cc = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t b[4];
            const int c = (2 * k + cc) & 7;
            ldsm4(kb0 + (k >> 2) * cstride + (n >> 1) * rstride + t * 128 + ((c ^ (t & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(s[mt][n], qf[mt][k], b[0], b[1]);
              mma_bf16(s[mt][n + 1], qf[mt][k], b[2], b[3]);
            }
          }
      }
      uint32_t p[MT][NT / 2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
          // Subtracted as integers: a position beyond 2^24 is no fp32 number.
          const float dist = (float)(pos[mt][e] - j0 - 2 * qc);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = j0 + 8 * n + 2 * qc + x;
              float v = s[mt][n][2 * e + x];
              if constexpr (MOD) {
                v *= a.scale;
                v = a.softcap > 0.0f ? a.softcap * tanh_log2e(v * a.inv_cap) : v * kLog2e;
                v = fmaf(-slope[mt][e], fabsf(dist - (float)(8 * n + x)), v);
              } else {
                v *= sl2;
              }
              v = j >= lo[mt][e] && j < hi[mt][e] ? v : -INFINITY;
              s[mt][n][2 * e + x] = v;
              top = fmaxf(top, v);
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float mn = fmaxf(m[mt][e], top);
          const float mu = mn == -INFINITY ? 0.0f : mn;
          if (__any_sync(0xffffffffu, mn > m[mt][e])) {
            const float f = ex2(m[mt][e] - mu);
            l[mt][e] *= f;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
              o[mt][n][2 * e] *= f;
              o[mt][n][2 * e + 1] *= f;
            }
            m[mt][e] = mn;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float p0 = ex2(s[mt][n][2 * e] - mu), p1 = ex2(s[mt][n][2 * e + 1] - mu);
            l[mt][e] += p0 + p1;
            // Rounded to bf16 for the second product only; the sum above
            // keeps the unrounded values.
            p[mt][n >> 1][2 * (n & 1) + e] = pack_bf16(p0, p1);
          }
        }
      if (!__all_sync(0xffffffffu, attn_wait(full + 8 * sv, ((done + 1) / kRing) & 1, status, kDevTimeoutFull, abort)))
        break;
      if (j0 < it_lo || j0 + KT > it_hi) {
        // Tokens that no row sees (never loaded, or the rest of a page): their
        // zero weights must not meet what lies there.
        for (int x = lane; x < KT * (DP / 8); x += 32) {
          const int t = x / (DP / 8), c = x % (DP / 8);
          if (j0 + t < it_lo || j0 + t >= it_hi)
            *reinterpret_cast<uint4 *>(ring + sv * C::kTile + (c >> 3) * cstride + (t >> 4) * rstride +
                                       (t & 15) * 128 + (((c & 7) ^ (t & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      {  // O += P V: matrix lane / 8 holds tokens 8 ((lane / 8) & 1), columns 8 (lane / 16)
        const int t = lane & 15, cc = lane >> 4;
#pragma unroll
        for (int k = 0; k < NT / 2; ++k)
#pragma unroll
          for (int n = 0; n < DP / 16; ++n) {
            uint32_t b[4];
            const int c = (2 * n + cc) & 7;
            ldsm4t(vb0 + (n >> 2) * cstride + k * rstride + t * 128 + ((c ^ (t & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(o[mt][2 * n], p[mt][k], b[0], b[1]);
              mma_bf16(o[mt][2 * n + 1], p[mt][k], b[2], b[3]);
            }
          }
      }
      // The tile's reads (and zeros) come before the copy that refills it.
      fence_proxy_async_smem();
      __syncwarp();
      done += 2;
      j0 += KT;
      --take;
    }
    // ---- the item's end
    if (take == 0) {
      const AttnSegment &g = segs[warp][popped % kSegs];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[mt][e];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          const int r = mt * 16 + e * 8 + qr, row = g.rb * R + r;
          if (row >= g.s.ql * a.G) continue;
          if (g.slot >= 0) {
            const int64_t at = (int64_t)g.slot * R + r;
            if (qc == 0) a.part_ml[at] = make_float2(m[mt][e], x);
            float *dst = a.part_o + at * DP + 2 * qc;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
              *reinterpret_cast<float2 *>(dst + 8 * n) = make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
            continue;
          }
          const AttnRow ar = attn_row(a, g.s, g.h, row);
          const AttnFinish f = attn_finish(a, ar, m[mt][e], x);
          if (qc == 0) attn_store_lse(a, f);
          const int64_t pat = f.id * DP + 2 * qc;
          if (a.prefix_pass) {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
              *reinterpret_cast<float2 *>(a.prev_o + pat + 8 * n) =
                  f.so == 0.0f ? make_float2(0.0f, 0.0f)
                               : make_float2(o[mt][n][2 * e] * f.so, o[mt][n][2 * e + 1] * f.so);
            continue;
          }
          const __nv_bfloat16 *gate = a.gate + ar.token * a.g_ts + ar.head * a.g_hs + 2 * qc;
          __nv_bfloat16 *dst = a.out + ar.token * a.o_ts + ar.head * a.o_hs + 2 * qc;
#pragma unroll
          for (int n0 = 0; n0 < DP / 8; n0 += 8) {
            uint32_t w[8];
            float2 q[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) {  // in flight together
              w[n] = 0u;
              q[n] = make_float2(0.0f, 0.0f);
              if (a.gate && 8 * (n0 + n) < a.D) w[n] = *reinterpret_cast<const uint32_t *>(gate + 8 * (n0 + n));
              if (a.prev_o && f.sp != 0.0f) q[n] = *reinterpret_cast<const float2 *>(a.prev_o + pat + 8 * (n0 + n));
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              float v0 = f.so == 0.0f ? 0.0f : o[mt][n0 + n][2 * e] * f.so;
              float v1 = f.so == 0.0f ? 0.0f : o[mt][n0 + n][2 * e + 1] * f.so;
              v0 = fmaf(q[n].x, f.sp, v0);
              v1 = fmaf(q[n].y, f.sp, v1);
              if (a.gate) {
                v0 *= sigmoidf(__uint_as_float(w[n] << 16));
                v1 *= sigmoidf(__uint_as_float(w[n] & 0xffff0000u));
              }
              if (8 * (n0 + n) < a.D) *reinterpret_cast<uint32_t *>(dst + 8 * (n0 + n)) = pack_bf16(v0, v1);
            }
          }
        }
      if (g.last_part >= 0 && lane == 0) a.meta[blockIdx.x * kWarps + warp] = attn_meta<R>(a, g);
      __syncwarp();
      ++popped;
      have = false;
    }
  }
  // Drain: the block never exits with a copy still writing its memory.
  for (; done < issued; ++done) {
    volatile int no_abort = 0;
    attn_wait(full + 8 * (done % kRing), (done / kRing) & 1, status, kDevTimeoutFull, &no_abort);
  }
}

template <int MT, int DP>
cudaError_t launch_rows(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int grid,
                        cudaStream_t st) {
  using C = RowsCfg<MT, DP>;
  const bool mod = a.softcap > 0.0f || a.slopes;
  auto k = mod ? attn_rows_kernel<MT, DP, true> : attn_rows_kernel<MT, DP, false>;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t e = attn_allow_smem(reinterpret_cast<const void *>(k), C::bytes, allowed[mod]);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = C::bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, k, tk, tv, a)) != cudaSuccess) return e;
  constexpr int RPB = 1;
  cfg.gridDim = dim3((unsigned)grid, (unsigned)(a.max_rows < C::R ? a.max_rows : C::R), (DP + 127) / 128);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attn_join_kernel<C::R, DP, kWarps, RPB>, a);
}

}  // namespace

cudaError_t launch_attn_rows(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int R,
                             int grid, cudaStream_t st) {
  if (a.D <= 64)
    return R == 16 ? launch_rows<1, 64>(tk, tv, a, grid, st) : launch_rows<2, 64>(tk, tv, a, grid, st);
  if (a.D <= 128) return launch_rows<1, 128>(tk, tv, a, grid, st);
  return launch_rows<1, 256>(tk, tv, a, grid, st);
}

int read_attn_rows_device_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_rows_status, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_attn_rows_status, &zero, sizeof(int));
  return v;
}

}  // namespace nvfp4
