// attention.cuh -- device side shared by the attention kernels
// (include/nvfp4_attention.h): the work of a call, its even division over the
// blocks of a launch, and the last step of a row.
//
// Query rows of one key/value head are laid out flat, row = token * G + query
// head within the group, so that the G heads that read a key share it.  An
// item is (sequence, key/value head, R consecutive rows); its keys, the union
// of what its rows see, are walked in units of KT.  All items' units, in the
// order sequence, head, rows, form one line of W units that the launch's
// blocks divide evenly: block c takes [c W / parts, (c + 1) W / parts).  An
// item cut by a block boundary leaves unnormalised parts in the workspace, at
// most two per block, which a second launch joins in the order of the blocks.
// The division depends on the lengths alone, so results repeat bit for bit.
#pragma once

#include <cuda_bf16.h>

#include "attention.h"

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

// An item that sees nothing still takes one unit of the line: its rows are
// written too.
template <int R, int KT>
__device__ __forceinline__ int attn_item_units(const AttnArgs &a, const AttnSeq &s, int rb) {
  return max(attn_item<R, KT>(a, s, rb).units, 1);
}

// Where a block starts on the line, and how far it goes.
struct AttnCursor {
  int b, h, rb, off;    // item and unit within it
  long long at, end;    // on the line
  long long total;      // W
  int parts;
};

struct AttnPlanSmem {
  int units[kPlanCache];  // per sequence and head
  long long sum[32];
  AttnCursor cur;
};

// Plans this block's share; every thread of the block calls it.  parts: at
// most gridDim.x and one per `min_units` units.
template <int R, int KT>
__device__ __forceinline__ AttnCursor attn_plan(const AttnArgs &a, int min_units, AttnPlanSmem *sm) {
  const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  const int NS = attn_num_seqs(a);
  long long sum = 0;
  // Sequences of few items: a thread each; of many: a warp each.
  const bool by_warp = a.max_blocks > 4;
  auto lane_units = [&](int b) -> int {  // by_warp: this lane's share
    const AttnSeq s = attn_seq(a, b);
    const int nb = attn_blocks<R>(a, s);
    int u = 0;
    for (int rb = by_warp ? lane : 0; rb < nb; rb += by_warp ? 32 : 1) u += attn_item_units<R, KT>(a, s, rb);
    return u;
  };
  auto warp_units = [&](int b) -> int {  // every lane gets sequence b's units
    int u = lane_units(b);
    if (by_warp)
      for (int o = 16; o; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    return u;
  };
  if (by_warp) {
    for (int b = warp; b < NS; b += nw) {
      const int u = warp_units(b);
      if (lane == 0) {
        if (b < kPlanCache) sm->units[b] = u;
        sum += u;
      }
    }
  } else {
    for (int b = tid; b < NS; b += nt) {
      const int u = lane_units(b);
      if (b < kPlanCache) sm->units[b] = u;
      sum += u;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sm->sum[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    long long total = 0;
    for (int i = 0; i < nw; ++i) total += sm->sum[i];
    total *= a.Hkv;
    AttnCursor c;
    c.total = total;
    const long long most = (total + min_units - 1) / min_units;
    c.parts = (int)(most < (long long)gridDim.x ? most : (long long)gridDim.x);
    c.b = c.h = c.rb = c.off = 0;
    c.at = c.end = 0;
    if ((int)blockIdx.x < c.parts) {
      c.at = (long long)blockIdx.x * total / c.parts;
      c.end = (long long)(blockIdx.x + 1) * total / c.parts;
      long long before = 0;
      long long o = c.at;
      int ub = 0;
      for (int base = 0; base < NS; base += 32) {  // the sequence that holds unit c.at
        long long u = 0;
        if (base + 32 <= kPlanCache || !by_warp) {
          const int b = base + lane;
          if (b < NS) u = b < kPlanCache ? sm->units[b] : lane_units(b);
        } else {
          for (int i = 0; i < 32 && base + i < NS; ++i) {
            const int w = warp_units(base + i);
            if (i == lane) u = w;
          }
        }
        long long inc = u * a.Hkv;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const long long v = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + inc > c.at);
        if (hit) {
          const int f = __ffs(hit) - 1;
          c.b = base + f;
          ub = (int)__shfl_sync(0xffffffffu, u, f);
          o = c.at - before - (__shfl_sync(0xffffffffu, inc, f) - (long long)ub * a.Hkv);
          break;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
      }
      c.h = (int)(o / ub);
      int r = (int)(o % ub);
      const AttnSeq s = attn_seq(a, c.b);
      const int nb = attn_blocks<R>(a, s);
      for (int base = 0; base < nb; base += 32) {  // the item within the sequence and head
        const int rb = base + lane;
        int inc = rb < nb ? attn_item_units<R, KT>(a, s, rb) : 0;
        const int u = inc;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > r);
        if (hit) {
          const int f = __ffs(hit) - 1;
          c.rb = base + f;
          c.off = r - (__shfl_sync(0xffffffffu, inc, f) - __shfl_sync(0xffffffffu, u, f));
          break;
        }
        r -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (lane == 0) sm->cur = c;
  }
  __syncthreads();
  return sm->cur;
}

// The next item on the line after (b, h, rb).
template <int R>
__device__ __forceinline__ void attn_next(const AttnArgs &a, AttnCursor &c, int nb) {
  c.off = 0;
  if (++c.rb < nb) return;
  c.rb = 0;
  if (++c.h < a.Hkv) return;
  c.h = 0;
  const int NS = attn_num_seqs(a);
  do {
    ++c.b;
  } while (c.b < NS && attn_seq(a, c.b).ql == 0);
}

// One stretch of a block's share: units [off, off + take) of an item.
struct AttnSegment {
  AttnSeq s;
  AttnItem it;
  int b, h, rb, off, take;
  bool whole;      // the block has all of the item
  int slot;        // workspace part otherwise
  bool leads;      // the item starts here and goes on in later blocks ...
  int last_part;   // ... up to this one
};

template <int R, int KT>
__device__ __forceinline__ bool attn_segment(const AttnArgs &a, AttnCursor &c, AttnSegment &g) {
  if (c.at >= c.end) return false;
  g.s = attn_seq(a, c.b);
  g.it = attn_item<R, KT>(a, g.s, c.rb);
  g.b = c.b;
  g.h = c.h;
  g.rb = c.rb;
  g.off = c.off;
  const int n = max(g.it.units, 1);
  const long long left = c.end - c.at;
  g.take = (int)(left < (long long)(n - c.off) ? left : (long long)(n - c.off));
  const bool ends = c.off + g.take == n;
  g.whole = c.off == 0 && ends;
  g.leads = c.off == 0 && !ends;
  g.slot = 2 * blockIdx.x + (g.leads ? 1 : 0);
  g.last_part = g.leads ? (int)(((c.at + n) * c.parts - 1) / c.total) : 0;
  c.at += g.take;
  c.off += g.take;
  if (ends) attn_next<R>(a, c, attn_blocks<R>(a, g.s));
  if (g.it.units == 0) g.take = 0;
  return true;
}

// The last step for 4 values of a row: o unnormalised against 2^m, l its sum.
// Joins the prefix pass's part, normalises, gates and stores (or, in the
// prefix pass, keeps the normalised row in fp32).
__device__ __forceinline__ void attn_finish4(const AttnArgs &a, const AttnRow &r, int d, int DP,
                                             float4 o, float m, float l) {
  if (d >= a.D) return;
  const int64_t rid = (int64_t)r.token * a.Hq + r.head;
  if (a.prefix_pass) {
    const float inv = l > 0.0f ? 1.0f / l : l != l ? l : 0.0f;
    *reinterpret_cast<float4 *>(a.prev_o + rid * DP + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (d == 0) a.prev_lse[rid] = l == 0.0f ? -INFINITY : m + log2f(l);
    return;
  }
  if (a.prev_o) {
    const float pl = a.prev_lse[rid];
    if (pl != -INFINITY) {
      const float top = fmaxf(m, pl);
      const float wo = m == -INFINITY ? 0.0f : exp2f(m - top), wp = exp2f(pl - top);
      const float4 p = *reinterpret_cast<const float4 *>(a.prev_o + rid * DP + d);
      o = make_float4(o.x * wo + p.x * wp, o.y * wo + p.y * wp, o.z * wo + p.z * wp, o.w * wo + p.w * wp);
      l = l * wo + wp;
      m = top;
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l != l ? l : 0.0f;
  float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  if (l == 0.0f) v[0] = v[1] = v[2] = v[3] = 0.0f;
  if (a.gate) {
    const uint2 g = *reinterpret_cast<const uint2 *>(a.gate + r.token * a.g_ts + r.head * a.g_hs + d);
    const float gv[4] = {__uint_as_float(g.x << 16), __uint_as_float(g.x & 0xffff0000u),
                         __uint_as_float(g.y << 16), __uint_as_float(g.y & 0xffff0000u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] / (1.0f + ex2(-gv[i] * kLog2e));
  }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2 *>(a.out + r.token * a.o_ts + r.head * a.o_hs + d) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
  if (d == 0 && a.lse) a.lse[rid] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
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
#pragma unroll
  for (int v = 0; v < V; ++v) attn_finish4(a, ar, 4 * lane + 128 * v, DP, acc[v], m, l);
}

}  // namespace nvfp4
