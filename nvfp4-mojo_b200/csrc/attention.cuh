// attention.cuh -- device side shared by the attention kernels
// (include/nvfp4_attention.h): the work of a call, its even division over the
// blocks of a launch, and the last step of a row.
//
// Query rows of one key/value head are laid out flat, row = token * G + query
// head within the group, so that the G heads that read a key share it.  An
// item is (sequence, key/value head, R consecutive rows); its keys, the union
// of what its rows see, are walked in units of KT.  All items' units, in the
// order sequence, head, rows, form one line of W units that the launch's
// blocks divide evenly: block c takes [c W / parts, (c + 1) W / parts).  W is
// below 2^31 (checked by the caller from the bounds of the call).  An
// item cut by a block boundary leaves unnormalised parts in the workspace, at
// most two per block, which a second launch joins in the order of the blocks.
// The division depends on the lengths alone, so results repeat bit for bit.
#pragma once

#include <cuda_bf16.h>

#include "attention.h"
#include "tc_common.cuh"

namespace nvfp4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPlanCache = 1024;  // sequences whose units the plan keeps in shared memory

struct AttnArgs {
  int B, T, Hq, Hkv, G, D;
  int page_size, page_shift, max_pages;
  int64_t pt_stride;
  const int *q_start, *kv_len, *page_table, *visible;
  int prefix_len;
  int prefix_pass;  // 1: all tokens against the shared prefix; 0: own keys
  int causal, window;
  int max_blocks;   // bound on items per sequence and head (max_q_len)
  float scale, softcap;
  const float *slopes;
  const __nv_bfloat16 *q, *gate;
  __nv_bfloat16 *out;
  int64_t q_ts, q_hs, g_ts, g_hs, o_ts, o_hs;
  float *lse;
  // Workspace: parts [2 * grid][R][DP] with their (max, sum), who joins what,
  // and the prefix pass's normalised rows [T, Hq, DP] with their lse (base 2).
  float *part_o;
  float2 *part_ml;
  int4 *meta;
  float *prev_o;
  float *prev_lse;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One sequence of a pass: its tokens, its keys in this pass and where the
// first token stands.
struct AttnSeq {
  int tok0, ql, n, pos0, vis;
};

__device__ __forceinline__ AttnSeq attn_own_seq(const AttnArgs &a, int b) {
  AttnSeq s;
  int e;
  if (a.q_start) {
    s.tok0 = min(max(a.q_start[b], 0), a.T);
    e = min(max(a.q_start[b + 1], s.tok0), a.T);
  } else {
    s.tok0 = b;
    e = b + 1;
  }
  s.ql = e - s.tok0;
  s.n = min(max(a.kv_len[b], 0), a.max_pages << a.page_shift);
  s.pos0 = a.prefix_len + s.n - s.ql;
  s.vis = a.visible ? a.visible[b] : 0;
  return s;
}

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b) {
  if (!a.prefix_pass) return attn_own_seq(a, b);
  return AttnSeq{0, a.T, a.prefix_len, 0, 0};
}

__device__ __forceinline__ int attn_num_seqs(const AttnArgs &a) { return a.prefix_pass ? 1 : a.B; }

// Keys [lo, hi) of the pass that the query at position p sees (hi <= lo: none).
__device__ __forceinline__ int2 attn_interval(const AttnArgs &a, int p, int vis, int n) {
  const int first = a.prefix_pass ? 0 : a.prefix_len;
  const int hi = a.causal ? min(max(p + 1, vis) - first, n) : n;
  const int lo = a.window > 0 ? max(p - a.window + 1 - first, 0) : 0;
  return make_int2(lo, hi);
}

// A row of an item: its token and head, position and keys.
struct AttnRow {
  int token, head, pos, lo, hi;
};

__device__ __forceinline__ AttnRow attn_row(const AttnArgs &a, const AttnSeq &s, int h, int row) {
  AttnRow r;
  const int i = row / a.G;
  r.head = h * a.G + (row - i * a.G);
  r.token = s.tok0 + i;
  r.lo = r.hi = 0;
  r.pos = 0;
  if (i >= s.ql) return r;
  if (!a.prefix_pass) {
    r.pos = s.pos0 + i;
    const int2 w = attn_interval(a, r.pos, s.vis, s.n);
    r.lo = w.x;
    r.hi = w.y;
  } else {
    // The token's own sequence: token t itself in a step of single tokens.
    int b = r.token;
    if (a.q_start) {
      b = min(b, a.B - 1);
      if (!(a.q_start[b] <= r.token && r.token < a.q_start[b + 1])) {
        int lo = 0, hi = a.B;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (a.q_start[mid + 1] > r.token) hi = mid;
          else lo = mid + 1;
        }
        b = lo;
        if (b >= a.B || a.q_start[b] > r.token) return r;  // in no sequence
      }
    }
    const AttnSeq o = attn_own_seq(a, b);
    r.pos = o.pos0 + r.token - o.tok0;
    const int2 w = attn_interval(a, r.pos, o.vis, s.n);
    r.lo = w.x;
    r.hi = w.y;
  }
  return r;
}

// The units of item `rb` of a sequence: first unit, count (0: its rows see
// nothing), and the keys [lo, hi) that any of its rows sees.
struct AttnItem {
  int u0, units, lo, hi;
};

template <int R, int KT>
__device__ __forceinline__ AttnItem attn_item(const AttnArgs &a, const AttnSeq &s, int rb) {
  AttnItem it;
  if (a.prefix_pass) {
    it.lo = 0;
    it.hi = s.n;
  } else {
    const int rows = s.ql * a.G;
    const int i0 = rb * R / a.G, i1 = (min((rb + 1) * R, rows) - 1) / a.G;
    it.lo = attn_interval(a, s.pos0 + i0, s.vis, s.n).x;
    it.hi = attn_interval(a, s.pos0 + i1, s.vis, s.n).y;
  }
  it.u0 = it.lo / KT;
  it.units = it.hi > it.lo ? (it.hi + KT - 1) / KT - it.u0 : 0;
  return it;
}

template <int R>
__device__ __forceinline__ int attn_blocks(const AttnArgs &a, const AttnSeq &s) {
  return (int)(((int64_t)s.ql * a.G + R - 1) / R);
}

// An item takes E more units of the line than it has, for what it costs to
// begin and end it (also where its rows see nothing: they are written too).
template <int R, int KT, int E>
__device__ __forceinline__ int attn_item_units(const AttnArgs &a, const AttnSeq &s, int rb) {
  return attn_item<R, KT>(a, s, rb).units + E;
}

// Bounded wait on an mbarrier phase, as mbar_wait (tc_common.cuh) in fewer
// instructions: the attention kernels wait in many places, and their code must
// stay in the instruction cache.
__device__ __forceinline__ bool attn_wait(uint32_t bar, uint32_t parity, int *status, int code,
                                          volatile int *abort) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    uint32_t t0, t;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t0));
    do {
      ok = mbar_try_wait(bar, parity);
      asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
      if (!ok && t - t0 > (uint32_t)kWaitLimitNs) {
        *status = code;
        *abort = 1;
      }
    } while (!ok && !*abort);
  }
  return ok;
}

// Where a block starts on the line, and how far it goes.
struct AttnCursor {
  int b, h, rb, off;  // item and unit within it
  int at, end;        // on the line
  int total, parts;   // W and the blocks that have a share
};

// The first unit of part c: floor(c total / parts).  The quotient's fraction
// is a multiple of 1 / parts, so a quarter unit before the division keeps the
// rounded product on the right side.
__device__ __forceinline__ int attn_line_at(int c, int total, int parts, double inv) {
  return (int)(((double)c * (double)total + 0.25) * inv);
}

struct AttnPlanSmem {
  int units[kPlanCache];  // per sequence and head
  int sum[32];
  AttnCursor cur;
};

// Plans this block's share; every thread of the block calls it.  parts: at
// most gridDim.x and one per `min_units` units.
template <int R, int KT, int E>
__device__ __forceinline__ AttnCursor attn_plan(const AttnArgs &a, int min_units, AttnPlanSmem *sm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int NS = attn_num_seqs(a);
  // Units of the items start, start + step, ... of sequence b and one head.
  auto seq_units = [&](int b, int start, int step) -> int {
    const AttnSeq s = attn_seq(a, b);
    const int nb = attn_blocks<R>(a, s);
    int u = 0;
#pragma unroll 1
    for (int rb = start; rb < nb; rb += step) u += attn_item_units<R, KT, E>(a, s, rb);
    return u;
  };
  // Sequences of few items: a thread each; of many: a warp each.
  const bool by_warp = a.max_blocks > 4;
  int sum = 0;
#pragma unroll 1
  for (int b = by_warp ? warp : tid; b < NS; b += by_warp ? nw : (int)blockDim.x) {
    int u = seq_units(b, by_warp ? lane : 0, by_warp ? 32 : 1);
    if (by_warp) u = __reduce_add_sync(0xffffffffu, u);
    if (!by_warp || lane == 0) {
      if (b < kPlanCache) sm->units[b] = u;
      sum += u;
    }
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (lane == 0) sm->sum[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    AttnCursor c = {};
    c.total = a.Hkv * __reduce_add_sync(0xffffffffu, lane < nw ? sm->sum[lane] : 0);
    c.parts = min((c.total + min_units - 1) / min_units, (int)gridDim.x);
    if ((int)blockIdx.x < c.parts) {
      const double inv = 1.0 / (double)c.parts;
      c.at = attn_line_at(blockIdx.x, c.total, c.parts, inv);
      c.end = attn_line_at(blockIdx.x + 1, c.total, c.parts, inv);
      // The sequence that holds unit c.at, 32 sequences at a time; then, with
      // its units per head, the item in the same way.
      int o = c.at, ub = 0;
#pragma unroll 1
      for (int base = 0; base < NS; base += 32) {
        const int b = base + lane;
        const int u = b >= NS ? 0 : b < kPlanCache ? sm->units[b] : seq_units(b, 0, 1);
        int inc = u * a.Hkv;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > o);
        if (hit) {
          const int f = __ffs(hit) - 1;
          c.b = base + f;
          ub = __shfl_sync(0xffffffffu, u, f);
          o -= __shfl_sync(0xffffffffu, inc, f) - ub * a.Hkv;
          break;
        }
        o -= __shfl_sync(0xffffffffu, inc, 31);
      }
      c.h = o / ub;
      o -= c.h * ub;
      const AttnSeq s = attn_seq(a, c.b);
      const int nb = attn_blocks<R>(a, s);
#pragma unroll 1
      for (int base = 0; base < nb; base += 32) {
        const int u = base + lane < nb ? attn_item_units<R, KT, E>(a, s, base + lane) : 0;
        int inc = u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > o);
        if (hit) {
          const int f = __ffs(hit) - 1;
          c.rb = base + f;
          c.off = o - (__shfl_sync(0xffffffffu, inc, f) - __shfl_sync(0xffffffffu, u, f));
          break;
        }
        o -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (lane == 0) sm->cur = c;
  }
  __syncthreads();
  return sm->cur;
}

// One stretch of a block's share: key units [off, off + take) of an item.
struct AttnSegment {
  AttnSeq s;
  AttnItem it;
  int b, h, rb, off, take;
  int slot;        // workspace part; -1: the block has all of the item
  int last_part;   // >= 0: the item starts here and goes on up to this block
};

template <int R, int KT, int E>
__device__ __forceinline__ bool attn_segment(const AttnArgs &a, AttnCursor &c, AttnSegment &g) {
#pragma unroll 1
  while (c.at < c.end) {
    g.s = attn_seq(a, c.b);
    const int nb = attn_blocks<R>(a, g.s);
    if (c.rb >= nb) {  // on to the next head or sequence
      c.rb = 0;
      if (nb == 0 || ++c.h == a.Hkv) {
        c.h = 0;
        ++c.b;
      }
      continue;
    }
    g.it = attn_item<R, KT>(a, g.s, c.rb);
    g.b = c.b;
    g.h = c.h;
    g.rb = c.rb;
    const int n = g.it.units + E, off = c.off;
    const int take = min(c.end - c.at, n - off);
    g.off = off;
    g.take = min(off + take, g.it.units) - min(off, g.it.units);
    const bool real = g.take > 0 || (g.it.units == 0 && off == 0);
    const bool first = off == 0, last = off + take >= g.it.units;
    g.slot = first && last ? -1 : 2 * (int)blockIdx.x + (first ? 1 : 0);
    g.last_part = -1;
    if (first && !last) {
      const int x = c.at + g.it.units - 1;  // the item's last unit
      const double inv = 1.0 / (double)c.parts;
      int p = min((int)((double)x * (double)c.parts / (double)c.total), c.parts - 1);
      while (p + 1 < c.parts && attn_line_at(p + 1, c.total, c.parts, inv) <= x) ++p;
      while (attn_line_at(p, c.total, c.parts, inv) > x) --p;
      g.last_part = p;
    }
    c.at += take;
    c.off += take;
    if (c.off == n) c.off = 0, ++c.rb;
    if (real) return true;
  }
  return false;
}

// The last step of a row: its output is o * so + prefix part * sp, gated.
struct AttnFinish {
  float so, sp, lse2;
  int64_t id;  // (token, head) of the row
};

// m, l: the row's maximum (base 2) and sum.
__device__ __forceinline__ AttnFinish attn_finish(const AttnArgs &a, const AttnRow &r, float m, float l) {
  AttnFinish f;
  f.id = (int64_t)r.token * a.Hq + r.head;
  f.sp = 0.0f;
  float w = 1.0f;
  if (a.prev_o && !a.prefix_pass) {
    const float pl = a.prev_lse[f.id];
    if (pl != -INFINITY) {
      const float top = fmaxf(m, pl);
      w = m == -INFINITY ? 0.0f : exp2f(m - top);
      f.sp = exp2f(pl - top);
      l = l * w + f.sp;
      m = top;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that sees nothing is 0
  f.so = w * inv;
  if (f.sp != 0.0f) f.sp *= inv;  // stays 0 without a prefix part, whatever l is
  f.lse2 = l == 0.0f ? -INFINITY : m + log2f(l);
  return f;
}

__device__ __forceinline__ void attn_store_lse(const AttnArgs &a, const AttnFinish &f) {
  if (a.prefix_pass) a.prev_lse[f.id] = f.lse2;
  else if (a.lse) a.lse[f.id] = f.lse2 * kLn2;
}

__device__ __forceinline__ float sigmoidf(float x) { return __fdividef(1.0f, 1.0f + ex2(-x * kLog2e)); }

// N = 4 or 8 values of the row from column d on (the prefix pass keeps the
// normalised row in fp32).
template <int N>
__device__ __forceinline__ void attn_store(const AttnArgs &a, const AttnRow &r, const AttnFinish &f, int d,
                                           int DP, float (&v)[N]) {
  if (d >= a.D) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = f.so == 0.0f ? 0.0f : v[i] * f.so;
  if (a.prefix_pass) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4 *>(a.prev_o + f.id * DP + d + i) =
          make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    return;
  }
  if (a.prev_o && f.sp != 0.0f) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 p = *reinterpret_cast<const float4 *>(a.prev_o + f.id * DP + d + i);
      v[i] = fmaf(p.x, f.sp, v[i]);
      v[i + 1] = fmaf(p.y, f.sp, v[i + 1]);
      v[i + 2] = fmaf(p.z, f.sp, v[i + 2]);
      v[i + 3] = fmaf(p.w, f.sp, v[i + 3]);
    }
  }
  if (a.gate) {
    const __nv_bfloat16 *gp = a.gate + r.token * a.g_ts + r.head * a.g_hs + d;
    uint32_t g[N / 2];
    if constexpr (N == 8) {
      const uint4 x = *reinterpret_cast<const uint4 *>(gp);
      g[0] = x.x, g[1] = x.y, g[2] = x.z, g[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2 *>(gp);
      g[0] = x.x, g[1] = x.y;
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      v[i] *= sigmoidf(__uint_as_float(g[i / 2] << 16));
      v[i + 1] *= sigmoidf(__uint_as_float(g[i / 2] & 0xffff0000u));
    }
  }
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
    w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
  }
  __nv_bfloat16 *op = a.out + r.token * a.o_ts + r.head * a.o_hs + d;
  if constexpr (N == 8) *reinterpret_cast<uint4 *>(op) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2 *>(op) = make_uint2(w[0], w[1]);
}

// Joins the parts of the items that blocks cut: blockIdx.x is the block that
// leads the item, a warp takes a row.
template <int R, int KT, int DP>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 w = a.meta[blockIdx.x];  // (sequence, head, rows, last part)
  if (w.w < 0) return;
  const AttnSeq s = attn_seq(a, w.x);
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int row = w.z * R + r;
  if (r >= R || row >= s.ql * a.G) return;
  const int c0 = blockIdx.x, np = w.w - c0 + 1;
  auto slot = [&](int i) -> int64_t { return i == 0 ? 2 * c0 + 1 : 2 * (c0 + i); };
  // The largest maximum and the joined sum, by the lanes over the parts.
  float m = -INFINITY;
  for (int i = lane; i < np; i += 32) m = fmaxf(m, a.part_ml[slot(i) * R + r].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  constexpr int V = DP >= 128 ? DP / 128 : 1;  // float4 per lane
  float4 acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int i = 0; i < np; ++i) {
    const float2 ml = a.part_ml[slot(i) * R + r];
    const float wt = ex2(ml.x - mu);
    l = fmaf(ml.y, wt, l);
    const float *o = a.part_o + (slot(i) * R + r) * DP;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int d = 4 * lane + 128 * v;
      if (d < DP) {
        const float4 x = *reinterpret_cast<const float4 *>(o + d);
        acc[v].x = fmaf(x.x, wt, acc[v].x);
        acc[v].y = fmaf(x.y, wt, acc[v].y);
        acc[v].z = fmaf(x.z, wt, acc[v].z);
        acc[v].w = fmaf(x.w, wt, acc[v].w);
      }
    }
  }
  const AttnRow ar = attn_row(a, s, w.y, row);
  const AttnFinish f = attn_finish(a, ar, m, l);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float x[4] = {acc[v].x, acc[v].y, acc[v].z, acc[v].w};
    attn_store<4>(a, ar, f, 4 * lane + 128 * v, DP, x);
  }
  if (lane == 0) attn_store_lse(a, f);
}

}  // namespace nvfp4
