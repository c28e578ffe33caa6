// attention.cuh -- device side shared by the attention kernels
// (include/nvfp4_attention.h): the work of a call, its even division over the
// blocks of a launch, and the last step of a row.
//
// Query rows of one key/value head are laid out flat, row = token * G + query
// head within the group, so that the G heads that read a key share it.  An
// item is (sequence, key/value head, R consecutive rows); its keys, the union
// of what its rows see, are walked in units of KT.  All items' units, in the
// order sequence, head, rows, form one line of W units that the launch's
// workers (blocks, or single warps) divide evenly: worker c takes
// [c W / parts, (c + 1) W / parts).  W is below 2^31 (checked by the caller from
// the bounds of the call).  An
// item cut by such a boundary leaves unnormalised parts in the workspace, at
// most two per worker, which a second launch joins in the order of the workers.
// The division depends on the lengths alone, so results repeat bit for bit.
#pragma once

#include <cuda_bf16.h>

#include "attention.h"
#include "tc_common.cuh"

namespace nvfp4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPlanCache = 1024;  // sequences whose units the plan keeps in shared memory

// What a worker leads: an item that starts in its share and goes on in later
// ones (last_part < 0: none).
struct __align__(16) AttnMeta {
  int last_part, tok0, h, row0;  // the item's first row (token * G + head) of its sequence
  int live, unused[3];           // its rows in use
};

struct AttnArgs {
  int B, T, Hq, Hkv, G, D;
  int page_size, page_shift, max_pages;
  int64_t pt_stride;
  const int *q_start, *kv_len, *page_table, *visible;
  int prefix_len;
  int prefix_pass;  // 1: all tokens against the shared prefix; 0: own keys
  int causal, window;
  int max_rows;     // of a sequence and key/value head, by max_q_len: sizes the
  int max_blocks;   // grid of the join; and their items: who plans
  int wide, wide_v; // a copy of keys (of values) brings all columns of its rows, not 64 of them
  float scale, softcap, inv_cap;
  const float *slopes;
  const __nv_bfloat16 *q, *gate;
  __nv_bfloat16 *out;
  int64_t q_ts, q_hs, g_ts, g_hs, o_ts, o_hs;
  float *lse;
  // Workspace: parts [2 * workers][R][DP] with their (max, sum), who joins what,
  // and the prefix pass's normalised rows [T, Hq, DP] with their lse (base 2).
  float *part_o;
  float2 *part_ml;
  AttnMeta *meta;
  float *prev_o;
  float *prev_lse;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2(e) tanh(x) = t P(t^2) / Q(t^2), t = x held to [-kTanhMax, kTanhMax]: the
// rational function of these degrees whose relative error on that interval is
// smallest (2.3e-8, from a weighted least-squares fit in 40 digits; tanh(kTanhMax)
// is 1 - 2.5e-8).  No coefficient is negative, so nothing cancels: evaluated in
// fp32 it is within 7 units of 2^-24 of the value at any x.  (cap - 2 cap / (1 +
// e^(2 x)) is off by 2^-22 of the cap, however small the score; with its two MUFU
// operations a score the three capped prompts of 28 / 4 heads of 128 took 145 us,
// with this one, more instructions and one MUFU operation, 146.)
constexpr float kTanhMax = 9.1f;
__device__ __forceinline__ constexpr float tanh_p(int k) {
  return k == 0   ? 1.442695022f
         : k == 1 ? 0.192951888f
         : k == 2 ? 0.00503172679f
         : k == 3 ? 2.95460250e-05f
                  : 1.90081302e-08f;
}
__device__ __forceinline__ constexpr float tanh_q(int k) {
  return k == 0   ? 1.0f
         : k == 1 ? 0.467077196f
         : k == 2 ? 0.0258470736f
         : k == 3 ? 0.000327278016f
                  : 7.70320810e-07f;
}

// The smaller of |x| and bound, with the sign of x; x where it is not a number.
__device__ __forceinline__ float hold(float x, float bound) {
  float y;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(bound));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tanh_log2e(float x) {
  const float t = hold(x, kTanhMax), u = t * t;
  float p = tanh_p(4), q = tanh_q(4);
#pragma unroll
  for (int k = 3; k >= 0; --k) {
    p = fmaf(p, u, tanh_p(k));
    q = fmaf(q, u, tanh_q(k));
  }
  return t * p * rcp(q);
}

// a / b for 0 <= a < 2^31, b > 0: the hardware's reciprocal, corrected (the
// plain quotient is several times as long, and much of a short call's time).
__device__ __forceinline__ int div_pos(int a, int b) {
  int q = (int)__fdividef((float)a, (float)b);
  int r = a - q * b;
  while (r < 0) --q, r += b;
  while (r >= b) ++q, r -= b;
  return q;
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
  const int i = div_pos(row, a.G);
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
    const int i0 = rb ? div_pos(rb * R, a.G) : 0, i1 = (rb + 1) * R < rows ? div_pos((rb + 1) * R - 1, a.G) : s.ql - 1;
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

// A box of the cache map into this block's shared memory: slots of one head and
// page, 64 columns from x on (or, wide, all of them, 64 columns after 64).
__device__ __forceinline__ void attn_load_box(uint32_t dst, const CUtensorMap *map, int x, int slot, int h, int page,
                                              uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7], %8;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(0), "r"(h), "r"(page), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ uint64_t l2_evict_normal_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
// Where a worker starts on the line, and how far it goes.
struct AttnCursor {
  int b, h, rb, off;  // item and unit within it
  int at, end;        // on the line
  int total, parts;   // W and the workers that have a share
  int worker;
};

// The first unit of part c: floor(c total / parts), in 32 bits (c and parts are
// at most a few hundred).
__device__ __forceinline__ int attn_line_at(int c, int total, int parts) {
  const int q = div_pos(total, parts), r = total - q * parts;
  return c * q + div_pos(c * r, parts);
}

struct AttnPlanSmem {
  int units[kPlanCache];  // per sequence and head
  int sum[32];
};

// Plans a worker's share; every thread of the block calls it.  Workers are the
// blocks (WARPS 0: the result is for warp `solo`, which lists the block's
// items), or the first WARPS warps of each.  parts: at most all workers and one
// per `min_units` units.
template <int R, int KT, int E, int WARPS>
__device__ __forceinline__ AttnCursor attn_plan(const AttnArgs &a, int min_units, AttnPlanSmem *sm, int solo) {
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
  // Sequences of few items: a thread each; of many: a warp each.  Of a few
  // sequences the warps that want a plan make it without the others.
  const bool by_warp = a.max_blocks > 4;
  const bool alone = NS <= (by_warp ? 4 : 32);
  if (alone && !WARPS && warp != solo) return AttnCursor{};
  int sum = 0;
#pragma unroll 1
  for (int b = by_warp ? (alone ? 0 : warp) : (alone ? lane : tid); b < NS;
       b += by_warp ? (alone ? 1 : nw) : (alone ? 32 : (int)blockDim.x)) {
    int u = seq_units(b, by_warp ? lane : 0, by_warp ? 32 : 1);
    if (by_warp) u = __reduce_add_sync(0xffffffffu, u);
    if (!by_warp || lane == 0) {
      if ((by_warp || !alone) && b < kPlanCache) sm->units[b] = u;  // (alone: each warp writes the same)
      sum += u;
    }
  }
  __syncwarp();
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (!alone) {
    if (lane == 0) sm->sum[warp] = sum;
    __syncthreads();
    sum = __reduce_add_sync(0xffffffffu, lane < nw ? sm->sum[lane] : 0);
  }
  AttnCursor c = {};
  if (WARPS ? warp < WARPS : warp == solo) {
    c.worker = WARPS ? blockIdx.x * WARPS + warp : blockIdx.x;
    c.total = a.Hkv * sum;
    c.parts = min(div_pos(c.total + min_units - 1, min_units), (int)gridDim.x * (WARPS ? WARPS : 1));
    if (c.worker < c.parts) {
      c.at = attn_line_at(c.worker, c.total, c.parts);
      c.end = attn_line_at(c.worker + 1, c.total, c.parts);
      // The sequence that holds unit c.at, 32 sequences at a time; then, with
      // its units per head, the item in the same way.
      int o = c.at, ub = 0;
      bool found = false;
#pragma unroll 1
      for (int base = 0; base < NS; base += 32) {
        const int b = base + lane;
        const int u = b >= NS ? 0 : (by_warp || !alone) && b < kPlanCache ? sm->units[b] : seq_units(b, 0, 1);
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
          found = true;
          break;
        }
        o -= __shfl_sync(0xffffffffu, inc, 31);
      }
      // Token ranges that overlap can make a longer line than the caller's bounds
      // allow for, and its length wrap: a place that is not on it is no work.
      found = found && o >= 0 && ub > 0;
      c.h = found ? div_pos(o, ub) : 0;
      found = found && c.h < a.Hkv;
      o -= c.h * ub;
      const AttnSeq s = attn_seq(a, c.b);
      const int nb = found ? attn_blocks<R>(a, s) : 0;
      found = false;
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
          found = true;
          break;
        }
        o -= __shfl_sync(0xffffffffu, inc, 31);
      }
      if (!found || c.off < 0) c.at = c.end;
    }
  }
  return c;
}

// One stretch of a worker's share: key units [off, off + take) of an item.
struct AttnSegment {
  AttnSeq s;
  AttnItem it;
  int b, h, rb, off, take;
  int slot;        // workspace part; -1: the worker has all of the item
  int last_part;   // >= 0: the item starts here and goes on up to this worker
};

template <int R, int KT, int E>
__device__ __forceinline__ bool attn_segment(const AttnArgs &a, AttnCursor &c, AttnSegment &g) {
#pragma unroll 1
  while (c.at < c.end) {
    if (c.b >= attn_num_seqs(a)) return false;  // (the line's end, see attn_plan)
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
    g.slot = first && last ? -1 : 2 * c.worker + (first ? 1 : 0);
    g.last_part = -1;
    if (first && !last) {
      const int x = c.at + g.it.units - 1;  // the item's last unit
      int p = min((int)__fdividef((float)x * (float)c.parts, (float)c.total), c.parts - 1);  // near it
#pragma unroll 1
      while (p + 1 < c.parts && attn_line_at(p + 1, c.total, c.parts) <= x) ++p;
#pragma unroll 1
      while (attn_line_at(p, c.total, c.parts) > x) --p;
      g.last_part = p;
    }
    c.at += take;
    c.off += take;
    if (c.off == n) c.off = 0, ++c.rb;
    if (real) return true;
  }
  return false;
}

template <int R>
__device__ __forceinline__ AttnMeta attn_meta(const AttnArgs &a, const AttnSegment &g) {
  AttnMeta m;
  m.last_part = g.last_part;
  m.tok0 = g.s.tok0;
  m.h = g.h;
  m.row0 = g.rb * R;
  m.live = min(g.s.ql * a.G - m.row0, R);
  return m;
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

// 4 values of the row from column d on (the prefix pass keeps the normalised
// row in fp32).
__device__ __forceinline__ void attn_store4(const AttnArgs &a, const AttnRow &r, const AttnFinish &f, int d,
                                            int DP, float (&v)[4]) {
  if (d >= a.D) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f.so == 0.0f ? 0.0f : v[i] * f.so;
  if (a.prefix_pass) {
    *reinterpret_cast<float4 *>(a.prev_o + f.id * DP + d) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
  if (a.prev_o && f.sp != 0.0f) {
    const float4 p = *reinterpret_cast<const float4 *>(a.prev_o + f.id * DP + d);
    v[0] = fmaf(p.x, f.sp, v[0]);
    v[1] = fmaf(p.y, f.sp, v[1]);
    v[2] = fmaf(p.z, f.sp, v[2]);
    v[3] = fmaf(p.w, f.sp, v[3]);
  }
  if (a.gate) {
    const uint2 g = *reinterpret_cast<const uint2 *>(a.gate + r.token * a.g_ts + r.head * a.g_hs + d);
    v[0] *= sigmoidf(__uint_as_float(g.x << 16));
    v[1] *= sigmoidf(__uint_as_float(g.x & 0xffff0000u));
    v[2] *= sigmoidf(__uint_as_float(g.y << 16));
    v[3] *= sigmoidf(__uint_as_float(g.y & 0xffff0000u));
  }
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2 *>(a.out + r.token * a.o_ts + r.head * a.o_hs + d) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}

// N columns' weighted sum of a row's parts, with their maximum and sum.
template <int V>
struct AttnParts {
  float m = -INFINITY, l = 0.0f;
  float4 acc[V] = {};
  __device__ __forceinline__ void add(float2 ml, const float4 (&x)[V]) {
    const float top = fmaxf(m, ml.x), mu = top == -INFINITY ? 0.0f : top;
    const float f = ex2(m - mu), g = ex2(ml.x - mu);
    m = top;
    l = l * f + ml.y * g;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      acc[v].x = acc[v].x * f + x[v].x * g;
      acc[v].y = acc[v].y * f + x[v].y * g;
      acc[v].z = acc[v].z * f + x[v].z * g;
      acc[v].w = acc[v].w * f + x[v].w * g;
    }
  }
  // Parts p, p + step, ... below np of row r of the item that worker c0 leads,
  // columns col + 128 v: IN of them in flight.
  template <int R, int DP, int IN>
  __device__ __forceinline__ void read(const AttnArgs &a, int c0, int r, int p, int step, int np, int col) {
#pragma unroll 1
    for (; p < np; p += IN * step) {
      float2 ml[IN];
      float4 x[IN][V];
#pragma unroll
      for (int q = 0; q < IN; ++q) {
        const int pp = min(p + q * step, np - 1);  // (a load that is not used, rather than a branch)
        const int64_t at = (int64_t)(pp == 0 ? 2 * c0 + 1 : 2 * (c0 + pp)) * R + r;
        ml[q] = a.part_ml[at];
#pragma unroll
        for (int v = 0; v < V; ++v)
          x[q][v] = *reinterpret_cast<const float4 *>(a.part_o + at * DP + min(col, DP - 4) + 128 * v);
      }
#pragma unroll
      for (int q = 0; q < IN; ++q)
        if (p + q * step < np) add(ml[q], x[q]);
    }
  }
};

__device__ __forceinline__ AttnRow attn_meta_row(const AttnArgs &a, const AttnMeta &w, int r) {
  AttnRow ar;
  const int t = div_pos(w.row0 + r, a.G);
  ar.token = w.tok0 + t;
  ar.head = w.h * a.G + w.row0 + r - t * a.G;
  return ar;
}

// Joins the parts of the items that workers cut.  A warp takes a row: with
// several rows per block (RPB, WPB 1) block (x, y) those from RPB y on of the
// item that worker x leads, else block (x, y) row y of the items that the
// workers 8 x .. 8 x + 7 lead, an item per warp.  There, items of seven parts and
// more come last: all eight warps take every eighth part, each block z 128
// columns, and join through shared memory.  Bound by latency: a part's loads
// depend on nothing but its place, so two, four or eight parts are in flight.
// (One context of 60000 keys, 592 parts a row: 53 us with four in flight per warp
// and one block per row, 43 so, attention included; prompts' items of 2 to 3 parts
// 276 us with two in flight, 287 with eight.  256 contexts of up to 400 keys: 55 us
// with one warp per block's items, 41 with one each.)
template <int R, int DP, int WPB, int RPB>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  static_assert((WPB == 1) != (RPB == 1) && (WPB == 1 || WPB == 8), "a warp's rows");
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int V = DP >= 128 ? DP / 128 : 1;  // float4 per lane
  const int last = a.meta[blockIdx.x * WPB + min(lane, WPB - 1)].last_part;
  const bool leads = lane < WPB && last >= 0, wide = RPB == 1 && last - (int)(blockIdx.x * WPB + lane) >= 6;
  if (blockIdx.z == 0 && __ballot_sync(0xffffffffu, leads && !wide && (WPB == 1 || lane == warp))) {
    const int c0 = blockIdx.x * WPB + (WPB == 1 ? 0 : warp);
    const AttnMeta w = a.meta[c0];
#pragma unroll 1
    for (int r = RPB * blockIdx.y + (WPB == 1 ? warp : 0); r < w.live; r += RPB * gridDim.y) {
      AttnParts<V> t;
      t.template read<R, DP, RPB == 1 ? 4 : 2>(a, c0, r, 0, 1, w.last_part - c0 + 1, 4 * lane);
      const AttnRow ar = attn_meta_row(a, w, r);
      const AttnFinish f = attn_finish(a, ar, t.m, t.l);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float x[4] = {t.acc[v].x, t.acc[v].y, t.acc[v].z, t.acc[v].w};
        attn_store4(a, ar, f, 4 * lane + 128 * v, DP, x);
      }
      if (lane == 0) attn_store_lse(a, f);
    }
  }
  if constexpr (RPB == 1) {
    __shared__ float4 s_o[8][32];
    __shared__ float2 s_ml[8];
    const int col = 128 * blockIdx.z + 4 * lane;
#pragma unroll 1
    for (unsigned todo = __ballot_sync(0xffffffffu, leads && wide); todo; todo &= todo - 1) {
      const int c0 = blockIdx.x * WPB + __ffs(todo) - 1;
      const AttnMeta w = a.meta[c0];
#pragma unroll 1
      for (int r = blockIdx.y; r < w.live; r += gridDim.y) {
        AttnParts<1> t;
        t.template read<R, DP, 8>(a, c0, r, warp, 8, w.last_part - c0 + 1, col);
        s_o[warp][lane] = t.acc[0];
        if (lane == 0) s_ml[warp] = make_float2(t.m, t.l);
        __syncthreads();
        if (warp == 0) {
#pragma unroll
          for (int q = 1; q < 8; ++q) {
            const float4 y[1] = {s_o[q][lane]};
            t.add(s_ml[q], y);
          }
          const AttnRow ar = attn_meta_row(a, w, r);
          const AttnFinish f = attn_finish(a, ar, t.m, t.l);
          float v[4] = {t.acc[0].x, t.acc[0].y, t.acc[0].z, t.acc[0].w};
          if (col < DP) attn_store4(a, ar, f, col, DP, v);
          if (col == 0) attn_store_lse(a, f);
        }
        __syncthreads();
      }
    }
  }
}

}  // namespace nvfp4
