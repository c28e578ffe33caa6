// attention_rows.cu -- attention of few query rows per key/value head (single
// tokens, a few tokens of speculative decoding) over the paged cache.
//
// Bound by HBM: every key and value is read once for the R = 16 or 32 rows
// that share it, in one launch whose blocks divide all sequences' keys evenly
// (attention.cuh), so a batch of ragged lengths keeps every SM streaming to
// the end.  One block per SM: a TMA producer warp keeps a ring of key and
// value tiles of 64 tokens in flight (a box per page, 128-byte swizzle), four
// warps each take 16 tokens of a tile: S = Q K^T and O += P V on mma.sync from
// registers (16 rows would fill an eighth of a tcgen05 tile), a softmax state
// (max, sum, O) per warp, no exchange between warps until the item ends.
#include <cuda_bf16.h>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention.cuh"
#include "attention_launch.h"
#include "tc_common.cuh"

namespace nvfp4 {

static __device__ int g_attn_rows_status;

namespace {

constexpr int kKT = 64;      // tokens per tile
constexpr int kWarps = 4;    // consumer warps, 16 tokens of a tile each
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kMergeBytes = 32768;
constexpr int kItemCost = 1;  // of an item's beginning and end, in tiles

template <int MT, int DP>
struct RowsCfg {
  static constexpr int R = 16 * MT;
  static constexpr int kTile = kKT * DP * 2;  // bytes of a key or value tile
  static constexpr int kMaxSlots = (227 * 1024 - kMergeBytes - 1024 - 8192) / kTile;
  static constexpr int kSlots = kMaxSlots > 16 ? 16 : kMaxSlots;
  static constexpr int MC = kMergeBytes / (kWarps * R * 4) < DP ? kMergeBytes / (kWarps * R * 4) : DP;
  static constexpr int offMerge = kSlots * kTile;
  static constexpr int bytes = offMerge + kMergeBytes + 1024;
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

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int h, int row,
                                            int page, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(row), "r"(page), "r"(bar), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void consumers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
}

// MOD: scores are capped or biased.
template <int MT, int DP, bool MOD>
__global__ void __launch_bounds__(kThreads, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ AttnArgs a) {
  using C = RowsCfg<MT, DP>;
  constexpr int R = C::R, kSlots = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  float *merge = reinterpret_cast<float *>(smem + C::offMerge);
  __shared__ AttnPlanSmem plan;
  __shared__ uint64_t bars[2 * 16];
  __shared__ float2 s_ml[kWarps][R];
  __shared__ int abort_flag;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full = smem_u32(bars), empty = full + 8 * 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kWarps);
    }
    mbar_fence_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  AttnCursor cur = attn_plan<R, kKT, kItemCost>(a, 1 + kItemCost, &plan);
  if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, -1);
  volatile int *abort = &abort_flag;
  AttnSegment g;

  if (warp == kWarps) {
    // ---------------- TMA producer ----------------
    const uint64_t policy = l2_evict_first_policy();
    const int box = a.page_size < kKT ? a.page_size : kKT;
    const int per = kKT / box;  // boxes (pages) per tile and 64 columns
    const int halves = DP / 64;
    int slot = 0, round = 0;
    bool ok = true;
    while (ok && attn_segment<R, kKT, kItemCost>(a, cur, g)) {
      const int *pages = a.page_table + (a.prefix_pass ? 0 : (int64_t)g.b * a.pt_stride);
      int ids = 0, ids_at = -64;
      for (int u = g.it.u0 + g.off; u < g.it.u0 + g.off + g.take && ok; ++u) {
        const int j0 = u * kKT;
        // This lane's box of the tile: rows j0 + i box .. of columns 64 hf.
        const int i = lane % per, hf = lane / per;
        const int tok = j0 + i * box;
        const bool mine = hf < halves && tok < g.it.hi && tok + box > g.it.lo;
        const int p0 = j0 >> a.page_shift, p1 = (j0 + kKT - 1) >> a.page_shift;
        if (p1 >= ids_at + 32 || p0 < ids_at) {  // the next 32 page ids, one per lane
          ids_at = p0;
          const int last = (g.it.hi - 1) >> a.page_shift;
          ids = pages[min(p0 + lane, last)];
        }
        const int page = __shfl_sync(0xffffffffu, ids, ((tok >> a.page_shift) - ids_at) & 31);
        const int row = tok & (a.page_size - 1);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * box * 128;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (round > 0) {
            const bool w = attn_wait(empty + 8 * slot, (round - 1) & 1, &g_attn_rows_status,
                                     kDevTimeoutEmpty, abort);
            if (!__all_sync(0xffffffffu, w)) {
              ok = false;
              break;
            }
          }
          if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, bytes);
          __syncwarp();
          if (mine)
            tma_load_4d(sbase + slot * C::kTile + hf * (kKT * 128) + i * box * 128, kv ? &tmV : &tmK,
                        64 * hf, g.h, row, page, full + 8 * slot, policy);
          if (++slot == kSlots) slot = 0, ++round;
        }
      }
    }
    // Drain: the block never exits with a copy still writing its memory.
    const int issued = round * kSlots + slot;
    for (int q = issued > kSlots ? issued - kSlots : 0; q < issued; ++q) {
      volatile int no_abort = 0;
      attn_wait(full + 8 * (q % kSlots), (q / kSlots) & 1, &g_attn_rows_status, kDevTimeoutFull, &no_abort);
    }
  } else {
    // ---------------- consumers ----------------
    const int qr = lane >> 2, qc = lane & 3;
    const float sl2 = a.scale * kLog2e;
    int slot = 0, round = 0;
    bool ok = true;
    while (ok && attn_segment<R, kKT, kItemCost>(a, cur, g)) {
      // Q fragments and the rows' key intervals.
      uint32_t qf[MT][DP / 16][4];
      int lo[MT][2], hi[MT][2], pos[MT][2];
      float slope[MT][2];
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
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int d = 16 * k + 8 * (x >> 1) + 2 * qc;
            qf[mt][k][x] = src[x & 1] && d < a.D ? src[x & 1][d >> 1] : 0u;
          }
      }
      float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        m[mt][0] = m[mt][1] = -INFINITY;
        l[mt][0] = l[mt][1] = 0.0f;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[mt][n][x] = 0.0f;
      }

      for (int u = g.it.u0 + g.off; u < g.it.u0 + g.off + g.take; ++u) {
        const int j0 = u * kKT + warp * 16;  // this warp's 16 tokens
        const bool any = j0 < g.it.hi && j0 + 16 > g.it.lo;
        float s[MT][2][4];
        // ---- S = Q K^T
        bool w = attn_wait(full + 8 * slot, round & 1, &g_attn_rows_status, kDevTimeoutFull, abort);
        if (!__all_sync(0xffffffffu, w)) {
          ok = false;
          break;
        }
        if (any) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 8; ++x) s[mt][x >> 2][x & 3] = 0.0f;
          // Matrix lane / 8: tokens 8 (lane / 16), columns 8 ((lane / 8) & 1).
          const int t = warp * 16 + (lane & 7) + 8 * (lane >> 4), cc = (lane >> 3) & 1;
          const uint32_t kb = sbase + slot * C::kTile + t * 128;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            uint32_t b[4];
            const int c = (2 * k + cc) & 7;
            ldsm4(kb + (k >> 2) * (kKT * 128) + ((c ^ (t & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(s[mt][0], qf[mt][k], b[0], b[1]);
              mma_bf16(s[mt][1], qf[mt][k], b[2], b[3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * slot);
        if (++slot == kSlots) slot = 0, ++round;
        // ---- softmax of this warp's 16 tokens
        uint32_t p[MT][4];
        if (any) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = -INFINITY;
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const int j = j0 + 8 * n + 2 * qc + x;
                  float v = s[mt][n][2 * e + x];
                  if constexpr (MOD) {
                    v *= a.scale;
                    if (a.softcap > 0.0f)  // cap tanh(v / cap)
                      v = a.softcap - __fdividef(2.0f * a.softcap, 1.0f + ex2(v * (2.0f * kLog2e / a.softcap)));
                    v = fmaf(v, kLog2e, -slope[mt][e] * fabsf((float)(pos[mt][e] - j)));
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
              for (int n = 0; n < 2; ++n) {
                const float p0 = ex2(s[mt][n][2 * e] - mu), p1 = ex2(s[mt][n][2 * e + 1] - mu);
                l[mt][e] += p0 + p1;
                // Rounded to bf16 for the second product only; the sum above
                // keeps the unrounded values.
                p[mt][2 * n + e] = pack_bf16(p0, p1);
              }
            }
          }
        }
        // ---- O += P V
        w = attn_wait(full + 8 * slot, round & 1, &g_attn_rows_status, kDevTimeoutFull, abort);
        if (!__all_sync(0xffffffffu, w)) {
          ok = false;
          break;
        }
        if (any) {
          const uint32_t vb0 = sbase + slot * C::kTile;
          if (j0 < g.it.lo || j0 + 16 > g.it.hi) {
            // Tokens that no row sees (never loaded, or the rest of a page):
            // their zero weights must not meet what lies there.
            for (int x = lane; x < 16 * (DP / 8); x += 32) {
              const int tt = warp * 16 + x / (DP / 8), j = j0 + x / (DP / 8), c = x % (DP / 8);
              if (j < g.it.lo || j >= g.it.hi)
                *reinterpret_cast<uint4 *>(smem + slot * C::kTile + (c >> 3) * (kKT * 128) + tt * 128 +
                                           (((c & 7) ^ (tt & 7)) << 4)) = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
          }
          // Matrix lane / 8: tokens 8 ((lane / 8) & 1), columns 8 (lane / 16).
          const int t = warp * 16 + (lane & 15), cc = lane >> 4;
          const uint32_t vb = vb0 + t * 128;
#pragma unroll
          for (int n = 0; n < DP / 16; ++n) {
            uint32_t b[4];
            const int c = (2 * n + cc) & 7;
            ldsm4t(vb + (n >> 2) * (kKT * 128) + ((c ^ (t & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(o[mt][2 * n], p[mt], b[0], b[1]);
              mma_bf16(o[mt][2 * n + 1], p[mt], b[2], b[3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * slot);
        if (++slot == kSlots) slot = 0, ++round;
      }
      if (!ok) break;

      // ---- the four warps' states joined, MC columns at a time
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[mt][e];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (qc == 0) s_ml[warp][mt * 16 + e * 8 + qr] = make_float2(m[mt][e], x);
        }
      constexpr int MC = C::MC;
#pragma unroll
      for (int c0 = 0; c0 < DP; c0 += MC) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < MC / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float2 *>(merge + (warp * R + mt * 16 + e * 8 + qr) * MC + 8 * n + 2 * qc) =
                  make_float2(o[mt][c0 / 8 + n][2 * e], o[mt][c0 / 8 + n][2 * e + 1]);
        consumers_sync();
        for (int x = threadIdx.x; x < R * (MC / 4); x += kWarps * 32) {
          const int r = x / (MC / 4), d = 4 * (x % (MC / 4));
          const int row = g.rb * R + r;
          if (row >= g.s.ql * a.G) continue;
          float mm = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_ml[w][r].x);
          const float mu = mm == -INFINITY ? 0.0f : mm;
          float ll = 0.0f;
          float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(s_ml[w][r].x - mu);
            ll = fmaf(s_ml[w][r].y, f, ll);
            const float4 v = *reinterpret_cast<const float4 *>(merge + (w * R + r) * MC + d);
            acc.x = fmaf(v.x, f, acc.x);
            acc.y = fmaf(v.y, f, acc.y);
            acc.z = fmaf(v.z, f, acc.z);
            acc.w = fmaf(v.w, f, acc.w);
          }
          if (g.slot < 0) {
            const AttnRow ar = attn_row(a, g.s, g.h, row);
            const AttnFinish f = attn_finish(a, ar, mm, ll);
            float x[4] = {acc.x, acc.y, acc.z, acc.w};
            attn_store<4>(a, ar, f, c0 + d, DP, x);
            if (c0 + d == 0) attn_store_lse(a, f);
          } else {
            *reinterpret_cast<float4 *>(a.part_o + ((int64_t)g.slot * R + r) * DP + c0 + d) = acc;
            if (c0 + d == 0) a.part_ml[(int64_t)g.slot * R + r] = make_float2(mm, ll);
          }
        }
        consumers_sync();
      }
      if (g.last_part >= 0 && threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(g.b, g.h, g.rb, g.last_part);
    }
  }
}

template <int MT, int DP>
cudaError_t launch_rows(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int grid,
                        cudaStream_t st) {
  using C = RowsCfg<MT, DP>;
  const bool mod = a.softcap > 0.0f || a.slopes;
  auto k = mod ? attn_rows_kernel<MT, DP, true> : attn_rows_kernel<MT, DP, false>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
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
  return cudaLaunchKernelEx(&cfg, attn_join_kernel<C::R, kKT, DP>, a);
}

}  // namespace

cudaError_t launch_attn_rows(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int R,
                             int grid, cudaStream_t st) {
  if (a.D <= 64)
    return R == 16 ? launch_rows<1, 64>(tk, tv, a, grid, st) : launch_rows<2, 64>(tk, tv, a, grid, st);
  if (a.D <= 128)
    return R == 16 ? launch_rows<1, 128>(tk, tv, a, grid, st) : launch_rows<2, 128>(tk, tv, a, grid, st);
  return launch_rows<1, 256>(tk, tv, a, grid, st);
}

int read_attn_rows_device_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_rows_status, sizeof(int)) != cudaSuccess) return -1;
  if (v) cudaMemcpyToSymbol(g_attn_rows_status, &zero, sizeof(int));
  return v;
}

}  // namespace nvfp4
