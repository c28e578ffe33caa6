// kv_append.cu -- appending keys and values to the paged cache, with the
// heads' norm and the position rotation on the way (include/nvfp4_attention.h).
//
// A row (one head of one token) belongs to a group of lanes of one warp, each
// holding 4 rotation pairs in registers; the group sums the squares for the
// norm by shuffles, turns its pairs and stores them.  A warp keeps its token's
// sines and cosines in registers and walks over that token's heads, so the
// angles (the only 64-bit arithmetic) are computed once per token and warp.
// Norm weight and rotation are one 2 x 2 matrix per pair, inv (x A - y B, y C +
// x E), and the rows ahead are loaded before the present ones are turned.  Bound
// by the issue of its instructions more than by HBM: 6424 tokens of 16 + 2 x 2
// heads of 256 take 37 us, 3.60 TB/s, at 160 instructions a row and 60 % of the
// issue slots.  (Three blocks per SM with four rows in flight per lane; two blocks,
// without spills, 41 us, four with two rows 47; products two at a time 35, but 40
// against 35 for 32 + 2 x 4 heads of 128.)  Latency-bound for a few tokens (64 of
// 32 + 2 x 4 heads of 128: 4.5 us): then a token's heads are spread over more warps,
// and the first rows' loads run under the angles.
#include <cuda_bf16.h>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention.h"
#include "kernels.h"

namespace nvfp4 {

int check_kv_cache(const nvfp4_kv_cache *c) {
  if (!c) return fail(NVFP4_ERR_INVALID_ARG, "null cache");
  if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 8)
    return fail(NVFP4_ERR_UNSUPPORTED, "head_dim %d: multiples of 8 up to 256", c->head_dim);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(NVFP4_ERR_UNSUPPORTED, "page_size %d: powers of two from 16 to 256", c->page_size);
  if (c->num_kv_heads <= 0 || c->num_kv_heads > 65535 || c->num_pages < 0 || c->num_pages > INT32_MAX)
    return fail(NVFP4_ERR_INVALID_ARG, "bad cache shape: %lld pages, %d heads", (long long)c->num_pages,
                c->num_kv_heads);
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] <= 0 || c->v_strides[i] <= 0 || c->k_strides[i] % 8 || c->v_strides[i] % 8 ||
        c->k_strides[i] >= (1ll << 38) || c->v_strides[i] >= (1ll << 38))
      return fail(NVFP4_ERR_INVALID_ARG, "cache strides must be positive multiples of 8 elements");
  if (c->num_pages > 0 && (!c->k || !c->v)) return fail(NVFP4_ERR_INVALID_ARG, "null cache pointer");
  if (!aligned(c->k, 16) || !aligned(c->v, 16))
    return fail(NVFP4_ERR_INVALID_ARG, "cache must be 16-byte aligned");
  return NVFP4_OK;
}

int check_attention_batch(const nvfp4_attention_batch *b, int page_size) {
  if (!b) return fail(NVFP4_ERR_INVALID_ARG, "null batch");
  if (b->num_seqs < 0 || b->num_seqs > (1 << 20) || b->num_tokens < 0 || b->num_tokens > (1 << 24) ||
      b->max_q_len < 0)
    return fail(NVFP4_ERR_INVALID_ARG, "bad batch: %d sequences, %lld tokens, max_q_len %d", b->num_seqs,
                (long long)b->num_tokens, b->max_q_len);
  if (!b->q_start && b->num_seqs != b->num_tokens)
    return fail(NVFP4_ERR_INVALID_ARG, "without q_start every sequence has one token: %d sequences, %lld tokens",
                b->num_seqs, (long long)b->num_tokens);
  if (b->num_tokens > 0 && b->num_seqs > 0 && b->max_q_len < 1)
    return fail(NVFP4_ERR_INVALID_ARG, "max_q_len %d with %lld tokens", b->max_q_len, (long long)b->num_tokens);
  if (b->prefix_len < 0 || b->max_pages < 0 ||
      (int64_t)b->max_pages * page_size + b->prefix_len + b->num_tokens > (1ll << 30))
    return fail(NVFP4_ERR_INVALID_ARG, "bad lengths: max_pages %d, prefix_len %d", b->max_pages, b->prefix_len);
  if (b->prefix_len > 0 && !b->prefix_pages) return fail(NVFP4_ERR_INVALID_ARG, "null prefix_pages");
  if (b->num_seqs > 0 && !b->kv_len) return fail(NVFP4_ERR_INVALID_ARG, "null kv_len");
  // (One row for all sequences is a stride of 0; of one sequence it means nothing.)
  if (b->num_seqs > 0 && b->max_pages > 0 &&
      (!b->page_table || (b->num_seqs > 1 && b->page_table_stride != 0 && b->page_table_stride < b->max_pages)))
    return fail(NVFP4_ERR_INVALID_ARG, "null page_table or stride below max_pages");
  return NVFP4_OK;
}

namespace {

constexpr int kAppendWarps = 8;

struct AppendArgs {
  nvfp4_kv_cache c;
  nvfp4_attention_batch b;
  nvfp4_rotary rot;  // rotary_dim 0: none
  nvfp4_qk_norm norm;
  nvfp4_head_rows q, k, v, qo;
  const int32_t *pos;
  int64_t pos_stride;
  int num_axes, num_heads, page_shift;
  int chunks;       // warps per token
  int chunk_steps;  // steps (of rows) per warp
};

__device__ __forceinline__ float bf(uint32_t w, int hi) {
  return __uint_as_float(hi ? (w & 0xffff0000u) : (w << 16));
}

// Four pairs as they lie in memory: runs of 4 consecutive elements from ei[0]
// and ej[0] on (HALVES), one run of 8 from ei[0] on (INTERLEAVED), or by element.
enum PairMode { kByElement = 0, kHalves = 1, kInterleaved = 2 };
template <typename T, int MODE>
struct RawPairs {
  static constexpr int N = sizeof(T) == 2 ? 4 : 8;
  uint32_t w[N];
  __device__ __forceinline__ void load(const T *row, const int (&ei)[4], const int (&ej)[4], bool on) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0u;
    if (!on) return;
    if constexpr (MODE != kByElement && sizeof(T) == 2) {
      if constexpr (MODE == kInterleaved) {
        const uint4 q = *reinterpret_cast<const uint4 *>(row + ei[0]);
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2 *>(row + ei[0]), y = *reinterpret_cast<const uint2 *>(row + ej[0]);
        w[0] = x.x, w[1] = x.y, w[2] = y.x, w[3] = y.y;
      }
    } else if constexpr (MODE != kByElement) {
      const uint4 x = *reinterpret_cast<const uint4 *>(row + ei[0]);
      const uint4 y = *reinterpret_cast<const uint4 *>(MODE == kInterleaved ? row + ei[0] + 4 : row + ej[0]);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
      w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          const uint16_t *r = reinterpret_cast<const uint16_t *>(row);
          w[i] = (ei[i] < 0 ? 0u : (uint32_t)r[ei[i]]) | (ej[i] < 0 ? 0u : (uint32_t)r[ej[i]]) << 16;
        } else {
          const uint32_t *r = reinterpret_cast<const uint32_t *>(row);
          w[i] = ei[i] < 0 ? 0u : r[ei[i]];
          w[4 + i] = ej[i] < 0 ? 0u : r[ej[i]];
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&a)[4], float (&b)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        constexpr bool side = MODE != kHalves;  // a pair in one word
        a[i] = side ? bf(w[i], 0) : bf(w[i >> 1], i & 1);
        b[i] = side ? bf(w[i], 1) : bf(w[2 + (i >> 1)], i & 1);
      } else {
        a[i] = __uint_as_float(MODE == kInterleaved ? w[2 * i] : w[i]);
        b[i] = __uint_as_float(MODE == kInterleaved ? w[2 * i + 1] : w[4 + i]);
      }
    }
  }
};

template <int MODE>
__device__ __forceinline__ void store_pairs(__nv_bfloat16 *row, const int (&ei)[4], const int (&ej)[4],
                                            const float (&a)[4], const float (&b)[4]) {
  constexpr bool inter = MODE == kInterleaved;
  if constexpr (MODE != kByElement) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = inter ? __floats2bfloat162_rn(a[i], b[i])
                               : i < 2 ? __floats2bfloat162_rn(a[2 * i], a[2 * i + 1])
                                       : __floats2bfloat162_rn(b[2 * i - 4], b[2 * i - 3]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    if constexpr (inter) {
      *reinterpret_cast<uint4 *>(row + ei[0]) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2 *>(row + ei[0]) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2 *>(row + ej[0]) = make_uint2(w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (ei[i] >= 0) row[ei[i]] = __float2bfloat16(a[i]);
      if (ej[i] >= 0) row[ej[i]] = __float2bfloat16(b[i]);
    }
  }
}

// LPR lanes per row (4 pairs each), 32 / LPR rows per warp step.
template <typename T, int LPR, int MODE>
__global__ void __launch_bounds__(kAppendWarps * 32, 3) kv_append_kernel(AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int RPW = 32 / LPR;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;  // rows a lane has in flight
  const int lane = threadIdx.x & 31, sub = lane / LPR, l = lane % LPR;
  const int64_t unit = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  const int64_t t = unit / a.chunks;
  if (t >= a.b.num_tokens) return;
  const int chunk = (int)(unit % a.chunks);

  // The token's sequence: token t itself in a step of single tokens (checked
  // first), else by bisection of q_start.
  int b = (int)t, qe = (int)t + 1;
  if (a.b.q_start) {
    const int B = a.b.num_seqs;
    b = min(b, B - 1);
    if (!(a.b.q_start[b] <= t && t < a.b.q_start[b + 1])) {
      int lo = 0, hi = B;  // the first b with q_start[b + 1] > t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.b.q_start[mid + 1] > t) hi = mid;
        else lo = mid + 1;
      }
      b = lo;
      if (b >= B || a.b.q_start[b] > t) return;  // in no sequence
    }
    qe = min(a.b.q_start[b + 1], (int)a.b.num_tokens);
  }
  const int64_t key = (int64_t)a.b.kv_len[b] - qe + t;  // own key index
  const int64_t at = key >> a.page_shift;
  int64_t page = -1;
  if (key >= 0 && at < a.b.max_pages) page = a.b.page_table[b * a.b.page_table_stride + at];
  const bool cached = page >= 0 && page < a.c.num_pages;
  const int slot = (int)(key & (a.c.page_size - 1));

  // This lane's pairs: p < rotary_dim / 2 are turned; the rest of the head is
  // paired half against half and only normed.
  const int D = a.c.head_dim, R = a.rot.rotary_dim, half = R / 2;
  const bool inter = MODE == kInterleaved || (MODE == kByElement && a.rot.interleaved);
  const bool active = l * 8 < D;
  int ei[4], ej[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = 4 * l + i;
    ei[i] = ej[i] = -1;
    if (2 * p < D) {
      if (inter) ei[i] = 2 * p, ej[i] = 2 * p + 1;
      else if (p < half) ei[i] = p, ej[i] = p + half;
      else ei[i] = R + (p - half), ej[i] = R + (p - half) + (D - R) / 2;
    }
  }

  // The token's rows in steps of RPW: heads of q, then of k, then of v, each
  // kind filled up to whole steps.  Pointers run along; they are worked out
  // anew only where the kind changes.
  const int HQ = a.num_heads, KV = a.c.num_kv_heads;
  const int sq = (HQ + RPW - 1) / RPW, sk = (KV + RPW - 1) / RPW;
  const int s0 = chunk * a.chunk_steps, s1 = min(sq + 2 * sk, s0 + a.chunk_steps);
  struct Run {
    int left, h, heads;  // steps of this kind left, this lane's head and their number
    int kind;
  };
  auto run_at = [&](int st) {
    Run r;
    r.kind = st < sq ? 0 : st < sq + sk ? 1 : 2;
    const int first = r.kind == 0 ? 0 : r.kind == 1 ? sq : sq + sk;
    r.left = (r.kind == 0 ? sq : sk) - (st - first);
    r.h = (st - first) * RPW + sub;
    r.heads = r.kind == 2 || r.kind == 1 ? KV : HQ;
    if (!active || (r.kind && !cached)) r.heads = 0;
    return r;
  };
  RawPairs<T, MODE> raw[kAhead];
  int fst = s0;  // the next step to fetch
  Run fr;
  fr.left = 0;
  const T *src = nullptr;
  int64_t sinc = 0;
  auto fetch = [&](RawPairs<T, MODE> &r) {
    if (fst >= s1) return;
    if (fr.left == 0) {
      fr = run_at(fst);
      const nvfp4_head_rows &in = fr.kind == 0 ? a.q : fr.kind == 1 ? a.k : a.v;
      src = static_cast<const T *>(in.data) + t * in.token_stride + fr.h * in.head_stride;
      sinc = RPW * in.head_stride;
    }
    r.load(src, ei, ej, fr.h < fr.heads);
    src += sinc;
    fr.h += RPW;
    --fr.left;
    ++fst;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(raw[i]);

  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = 4 * l + i;
    cs[i] = 1.0f, sn[i] = 0.0f;
    if (p < half) {
      int axis = a.rot.axis ? a.rot.axis[p] : 0;
      axis = axis < 0 ? 0 : axis >= a.num_axes ? a.num_axes - 1 : axis;
      const int64_t pos = a.pos ? a.pos[axis * a.pos_stride + t] : key + a.b.prefix_len;
      // Whole turns are taken off in 64 bits: pos * inv_freq / (2 pi) keeps
      // 2^-53 of up to 2^31 turns, far below fp32's step of the remainder.
      const double turns = (double)pos * (double)a.rot.inv_freq[p] * 0.15915494309189533577;
      sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
      cs[i] *= a.rot.scale;
      sn[i] *= a.rot.scale;
    }
  }

  const float inv_d = 1.0f / (float)D;
  float A[4], B[4], C[4], E[4];  // x' = x A - y B, y' = y C + x E
  Run wr;
  wr.left = 0;
  wr.kind = 0;
  bool normed = false;
  __nv_bfloat16 *dst = nullptr;
  int64_t dinc = 0;
#pragma unroll 1
  for (int sb = s0; sb < s1; sb += kAhead)
#pragma unroll
    for (int ring = 0; ring < kAhead; ++ring) {
      const int st = sb + ring;
      if (st >= s1) break;
      if (wr.left == 0) {
        wr = run_at(st);
        const __nv_bfloat16 *w = static_cast<const __nv_bfloat16 *>(wr.kind == 0   ? a.norm.q_weight
                                                                    : wr.kind == 1 ? a.norm.k_weight
                                                                                   : nullptr);
        normed = w != nullptr;
        float wx[4], wy[4];
        RawPairs<__nv_bfloat16, MODE> rw;
        rw.load(w, ei, ej, normed && active);
        rw.get(wx, wy);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = normed ? wx[i] + a.norm.weight_offset : 1.0f, q = normed ? wy[i] + a.norm.weight_offset : 1.0f;
          A[i] = p * cs[i], B[i] = q * sn[i], C[i] = q * cs[i], E[i] = p * sn[i];
        }
        if (wr.kind == 0) {
          dst = static_cast<__nv_bfloat16 *>(a.qo.data) + t * a.qo.token_stride + wr.h * a.qo.head_stride;
          dinc = RPW * a.qo.head_stride;
        } else {
          const int64_t *cstr = wr.kind == 1 ? a.c.k_strides : a.c.v_strides;
          dst = static_cast<__nv_bfloat16 *>(wr.kind == 1 ? a.c.k : a.c.v) + page * cstr[0] + slot * cstr[1] +
                wr.h * cstr[2];
          dinc = RPW * cstr[2];
        }
      }
      float x[4], y[4];
      raw[ring].get(x, y);
      fetch(raw[ring]);
      float inv = 1.0f;
      if (normed) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(x[i], x[i], fmaf(y[i], y[i], s));
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        inv = rsqrtf(s * inv_d + a.norm.eps);
      }
      if (wr.kind < 2) {  // values pass as they are, whatever they are
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (A pair that is not turned has no product with its partner, which may be infinite.)
          float u = x[i] * A[i], v = y[i] * C[i];
          if (4 * l + (MODE == kHalves ? 0 : i) < half) {  // (halves: four pairs alike)
            u = fmaf(-y[i], B[i], u);
            v = fmaf(x[i], E[i], v);
          }
          x[i] = u * inv, y[i] = v * inv;
        }
      }
      if (wr.h < wr.heads) store_pairs<MODE>(dst, ei, ej, x, y);
      dst += dinc;
      wr.h += RPW;
      --wr.left;
    }
}

template <typename T, int LPR>
cudaError_t launch_append(AppendArgs &a, bool vec, cudaStream_t st) {
  constexpr int RPW = 32 / LPR;
  const int steps = (a.num_heads + RPW - 1) / RPW + 2 * ((a.c.num_kv_heads + RPW - 1) / RPW);
  // A warp takes a whole token where there are tokens enough for 16 warps on
  // every SM; fewer tokens are split over up to one warp per step of rows.
  // (400 tokens of 32 + 2 x 4 heads of 128: 7.9 us for 4 warps, 6.2 for 16, 7.9 for
  // 48; 1500 tokens 14.1, 10.3, 14.1; 64 tokens 4.2, 4.5, 4.5.)
  const int64_t want = (int64_t)attn_sms() * 16;
  int64_t chunks = a.b.num_tokens >= want ? 1 : (want + a.b.num_tokens - 1) / a.b.num_tokens;
  if (chunks > steps) chunks = steps;
  a.chunk_steps = (int)((steps + chunks - 1) / chunks);
  a.chunks = (steps + a.chunk_steps - 1) / a.chunk_steps;
  const int64_t warps = a.b.num_tokens * a.chunks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((warps + kAppendWarps - 1) / kAppendWarps), 1, 1);
  cfg.blockDim = dim3(kAppendWarps * 32, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return !vec                ? cudaLaunchKernelEx(&cfg, kv_append_kernel<T, LPR, kByElement>, a)
         : a.rot.interleaved ? cudaLaunchKernelEx(&cfg, kv_append_kernel<T, LPR, kInterleaved>, a)
                             : cudaLaunchKernelEx(&cfg, kv_append_kernel<T, LPR, kHalves>, a);
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_kv_append(const nvfp4_kv_cache *cache, const nvfp4_attention_batch *batch,
                               const nvfp4_rotary *rotary, const nvfp4_qk_norm *norm,
                               const nvfp4_head_rows *q, const nvfp4_head_rows *k,
                               const nvfp4_head_rows *v, int in_dtype, int32_t num_heads,
                               const int32_t *positions, int64_t position_stride, int32_t num_axes,
                               const nvfp4_head_rows *q_out, void *stream) {
  NVFP4_ABI_RANGE();
  int rc = check_kv_cache(cache);
  if (rc) return rc;
  if ((rc = check_attention_batch(batch, cache->page_size))) return rc;
  if (in_dtype != NVFP4_DTYPE_F32 && in_dtype != NVFP4_DTYPE_BF16)
    return fail(NVFP4_ERR_INVALID_ARG, "bad dtype");
  if (num_heads <= 0 || num_heads > 65535) return fail(NVFP4_ERR_INVALID_ARG, "bad num_heads %d", num_heads);
  if (!q || !k || !v || !q_out) return fail(NVFP4_ERR_INVALID_ARG, "null row descriptor");
  const int R = rotary ? rotary->rotary_dim : 0;
  if (rotary && (R <= 0 || R % 2 || R > cache->head_dim || !rotary->inv_freq))
    return fail(NVFP4_ERR_INVALID_ARG, "rotary_dim %d: even, 2 .. head_dim, with inv_freq", R);
  if (positions &&
      (num_axes < 1 || (num_axes > 1 && position_stride != 0 && position_stride < batch->num_tokens)))
    return fail(NVFP4_ERR_INVALID_ARG, "positions need num_axes >= 1 rows of num_tokens");
  if (norm && !(norm->eps >= 0.0f)) return fail(NVFP4_ERR_INVALID_ARG, "eps must not be negative");
  if (batch->num_tokens == 0 || batch->num_seqs == 0) return NVFP4_OK;
  if (!q->data || !k->data || !v->data || !q_out->data) return fail(NVFP4_ERR_INVALID_ARG, "null row pointer");
  const int esize = in_dtype == NVFP4_DTYPE_BF16 ? 2 : 4;
  if (q->data == q_out->data &&
      (esize != 2 || q->token_stride != q_out->token_stride || q->head_stride != q_out->head_stride))
    return fail(NVFP4_ERR_INVALID_ARG, "q_out is q with another dtype or stride");
  // Rows are written while others are still read: in their own places only.
  auto span = [&](const nvfp4_head_rows *r, int heads, int es) {
    return head_span(*r, batch->num_tokens, heads, cache->head_dim, es);
  };
  const RowSpan so = span(q_out, num_heads, 2), sq = span(q, num_heads, esize);
  if (rows_overlap(so)) return fail(NVFP4_ERR_INVALID_ARG, "rows of q_out overlap");
  if ((!same_rows(so, sq) && rows_overlap(so, sq)) || rows_overlap(so, span(k, cache->num_kv_heads, esize)) ||
      rows_overlap(so, span(v, cache->num_kv_heads, esize)))
    return fail(NVFP4_ERR_INVALID_ARG, "q_out overlaps k, v, or q in other places than its own");
  if (cache->num_pages > 0 && cache->k == cache->v)
    return fail(NVFP4_ERR_INVALID_ARG, "keys and values share their places in the cache");
  AppendArgs a = {};
  a.c = *cache;
  a.b = *batch;
  if (rotary) a.rot = *rotary;
  if (norm) a.norm = *norm;
  a.q = *q;
  a.k = *k;
  a.v = *v;
  a.qo = *q_out;
  a.pos = positions;
  a.pos_stride = position_stride;
  a.num_axes = positions ? num_axes : 1;
  a.num_heads = num_heads;
  for (a.page_shift = 4; (1 << a.page_shift) < cache->page_size;) ++a.page_shift;
  // Runs of 4 pairs as 8- or 16-byte accesses: the halves of the turned and
  // of the plain part must hold whole runs, on aligned rows.
  const int D = cache->head_dim;
  auto fits = [&](const nvfp4_head_rows *r, int es) {
    return aligned(r->data, 16) && (r->token_stride * es) % 16 == 0 && (r->head_stride * es) % 16 == 0;
  };
  const bool vec = fits(q, esize) && fits(k, esize) && fits(v, esize) && fits(q_out, 2) &&
                   aligned(a.norm.q_weight, 16) && aligned(a.norm.k_weight, 16) &&
                   (a.rot.interleaved || (R % 8 == 0 && (D - R) % 8 == 0));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (in_dtype == NVFP4_DTYPE_BF16)
    e = D <= 64 ? launch_append<__nv_bfloat16, 8>(a, vec, st)
        : D <= 128 ? launch_append<__nv_bfloat16, 16>(a, vec, st)
                   : launch_append<__nv_bfloat16, 32>(a, vec, st);
  else
    e = D <= 64 ? launch_append<float, 8>(a, vec, st)
        : D <= 128 ? launch_append<float, 16>(a, vec, st)
                   : launch_append<float, 32>(a, vec, st);
  return check_launch(e, "cache append launch");
}
