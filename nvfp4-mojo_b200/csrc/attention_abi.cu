// attention_abi.cu -- nvfp4_paged_attention: checks, the workspace's layout
// and the passes (include/nvfp4_attention.h).
#include <atomic>
#include <cfloat>
#include <cmath>

#include "../../include/nvfp4.h"
#include "abi_util.h"
#include "attention_launch.h"
#include "kernels.h"

namespace nvfp4 {

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);

static EncodeFn attn_encode() {
  static EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// (column, slot, 64-column block, head, page) of the keys or values, boxes of 64
// columns by `rows` slots of one head and page: all blocks of columns at once
// (wide), or one, with the columns beyond the head reading as zeros.
static bool make_cache_map(CUtensorMap *m, void *base, const int64_t (&st)[3], const nvfp4_kv_cache &c, int rows,
                           bool wide) {
  EncodeFn fn = attn_encode();
  if (!fn) return false;
  const cuuint64_t blocks = wide ? c.head_dim / 64 : 1;
  cuuint64_t dims[5] = {wide ? 64 : (cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, blocks,
                        (cuuint64_t)c.num_kv_heads, (cuuint64_t)c.num_pages};
  cuuint64_t strides[4] = {(cuuint64_t)st[1] * 2, 128, (cuuint64_t)st[2] * 2, (cuuint64_t)st[0] * 2};
  cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)blocks, 1, 1};
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, base, dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attn_sms() {
  static std::atomic<int> count[64];  // per device
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if ((n = count[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  count[dev].store(n, std::memory_order_relaxed);
  return n;
}

cudaError_t attn_allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> &devices) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (devices.load(std::memory_order_relaxed) >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) devices.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

namespace {

int check_desc(const nvfp4_attention_desc *d) {
  if (!d) return fail(NVFP4_ERR_INVALID_ARG, "null attention descriptor");
  if (d->num_heads <= 0 || d->num_kv_heads <= 0 || d->num_heads > 65535 || d->num_heads % d->num_kv_heads)
    return fail(NVFP4_ERR_INVALID_ARG, "num_heads %d must be a multiple of num_kv_heads %d", d->num_heads,
                d->num_kv_heads);
  if (d->num_heads / d->num_kv_heads > 128)
    return fail(NVFP4_ERR_UNSUPPORTED, "more than 128 query heads per key/value head");
  if (d->head_dim <= 0 || d->head_dim > 256 || d->head_dim % 8)
    return fail(NVFP4_ERR_UNSUPPORTED, "head_dim %d: multiples of 8 up to 256", d->head_dim);
  if (!std::isfinite(d->scale) || !(d->scale > 0.0f) || !std::isfinite(d->softcap) || d->softcap < 0.0f)
    return fail(NVFP4_ERR_INVALID_ARG, "scale must be positive, softcap not negative, both finite");
  if (d->window < 0) return fail(NVFP4_ERR_INVALID_ARG, "window must not be negative");
  return NVFP4_OK;
}

// Query rows of an item, which also names the kernel: 16, or 32 at head sizes up
// to 64, on attention_rows.cu while a sequence's rows per key/value head fit one
// item, else attention_tc.cu.  Measured on the one and on the other, 64 sequences
// of 200 to 12000 keys, 4 key/value heads: 8 rows of 128 133 and 174 us (256
// sequences of up to 400 keys 41 and 81), 24 to 32 rows of 128 211 and 166 us, of
// 64 114 and 157 us; 33 rows and more, whose keys attention_rows.cu would read
// twice, 394 and 175 us.
int rows_of(const nvfp4_attention_desc &d, int64_t rows) {
  if (rows <= 16) return 16;
  if (d.head_dim > 128) return 128;
  return rows <= 32 && d.head_dim <= 64 ? 32 : 256;
}

struct AttnLayout {
  size_t part_o, part_ml, meta, prev_o, prev_lse, total;
  int dp, R0, R1;  // rows per item of the prefix pass and of the own pass
};

AttnLayout attn_layout(const nvfp4_attention_desc &d, const nvfp4_attention_batch &b, int grid) {
  AttnLayout L;
  const int G = d.num_heads / d.num_kv_heads;
  L.dp = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256;
  L.R1 = rows_of(d, (int64_t)b.max_q_len * G);
  L.R0 = b.prefix_len > 0 ? rows_of(d, b.num_tokens * G) : 0;
  // Rows of parts: two per worker, of the larger pass.
  auto part_rows = [&](int R) -> size_t { return (size_t)2 * grid * R * (R <= 32 ? kAttnRowsWorkers : 1); };
  const size_t rows = part_rows(L.R0) > part_rows(L.R1) ? part_rows(L.R0) : part_rows(L.R1);
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  size_t at = 0;
  L.part_o = at;
  at += up(rows * L.dp * 4);
  L.part_ml = at;
  at += up(rows * 8);
  L.meta = at;
  at += up((size_t)grid * kAttnRowsWorkers * sizeof(AttnMeta));
  L.prev_o = at;
  if (b.prefix_len > 0) at += up((size_t)b.num_tokens * d.num_heads * L.dp * 4);
  L.prev_lse = at;
  if (b.prefix_len > 0) at += up((size_t)b.num_tokens * d.num_heads * 4);
  L.total = at;
  return L;
}

// The line of units (attention.cuh) is counted in 31 bits.
int check_size(const nvfp4_attention_desc &d, const nvfp4_attention_batch &b, int page_size) {
  const int64_t G = d.num_heads / d.num_kv_heads;
  const double keys = (double)b.max_pages * page_size, rows = (double)b.num_tokens * G;
  const AttnLayout L = attn_layout(d, b, 1);
  auto line = [&](int R, double n, double seqs) {
    return d.num_kv_heads * (rows / R + seqs) * (n / (R <= 32 ? attn_rows_tile(d.head_dim) : 64) + 8);
  };
  if (rows >= (double)(1ll << 30) || line(L.R1, keys, b.num_seqs) >= 2147483648.0 ||
      (b.prefix_len > 0 && line(L.R0, b.prefix_len, 1) >= 2147483648.0))
    return fail(NVFP4_ERR_UNSUPPORTED, "%lld tokens against up to %.0f keys in one call",
                (long long)b.num_tokens, keys + b.prefix_len);
  return NVFP4_OK;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" size_t nvfp4_attention_workspace_size(const nvfp4_attention_desc *desc,
                                                 const nvfp4_attention_batch *batch) {
  if (check_desc(desc) || check_attention_batch(batch, 16)) return 0;
  return attn_layout(*desc, *batch, attn_sms()).total;
}

extern "C" int nvfp4_paged_attention(const nvfp4_attention_desc *desc, const nvfp4_head_rows *q,
                                     const nvfp4_kv_cache *cache, const nvfp4_attention_batch *batch,
                                     const float *slopes, const nvfp4_head_rows *gate,
                                     const nvfp4_head_rows *out, float *lse, void *ws, size_t ws_bytes,
                                     void *stream) {
  NVFP4_ABI_RANGE();
  int rc = check_desc(desc);
  if (rc) return rc;
  if ((rc = check_kv_cache(cache))) return rc;
  if ((rc = check_attention_batch(batch, cache->page_size))) return rc;
  if (cache->num_kv_heads != desc->num_kv_heads || cache->head_dim != desc->head_dim)
    return fail(NVFP4_ERR_INVALID_ARG, "cache has %d heads of %d, descriptor %d of %d", cache->num_kv_heads,
                cache->head_dim, desc->num_kv_heads, desc->head_dim);
  if ((rc = check_size(*desc, *batch, cache->page_size))) return rc;
  if (!q || !out) return fail(NVFP4_ERR_INVALID_ARG, "null row descriptor");
  if (batch->num_tokens == 0 || batch->num_seqs == 0) return NVFP4_OK;
  if (cache->num_pages <= 0) return fail(NVFP4_ERR_INVALID_ARG, "cache without pages");
  auto rows_ok = [](const nvfp4_head_rows *r) {
    return r->data && aligned(r->data, 16) && r->token_stride % 8 == 0 && r->head_stride % 8 == 0;
  };
  if (!rows_ok(q) || !rows_ok(out) || (gate && !rows_ok(gate)))
    return fail(NVFP4_ERR_INVALID_ARG,
                "q, out and gate: not null, 16-byte aligned, strides multiples of 8 elements");
  if (q->data == out->data && (q->token_stride != out->token_stride || q->head_stride != out->head_stride))
    return fail(NVFP4_ERR_INVALID_ARG, "out is q with another stride");
  // Rows are written while others are still read: in their own places only.
  auto span = [&](const nvfp4_head_rows *r) {
    return head_span(*r, batch->num_tokens, desc->num_heads, desc->head_dim, 2);
  };
  const RowSpan so = span(out), sq = span(q);
  if (rows_overlap(so)) return fail(NVFP4_ERR_INVALID_ARG, "rows of out overlap");
  if ((!same_rows(so, sq) && rows_overlap(so, sq)) || (gate && !same_rows(so, span(gate)) && rows_overlap(so, span(gate))))
    return fail(NVFP4_ERR_INVALID_ARG, "out overlaps q or gate in other places than its own");
  if (lse) {
    const RowSpan sl = {lse, (int64_t)batch->num_tokens * desc->num_heads * 4, {1, 1}, {0, 0}};
    if (rows_overlap(sl, so) || rows_overlap(sl, sq) || (gate && rows_overlap(sl, span(gate))))
      return fail(NVFP4_ERR_INVALID_ARG, "lse overlaps q, gate or out");
  }
  const int grid = attn_sms();
  const AttnLayout L = attn_layout(*desc, *batch, grid);
  if (!ws || !aligned(ws, 256)) return fail(NVFP4_ERR_INVALID_ARG, "null workspace or not 256-byte aligned");
  if (ws_bytes < L.total)
    return fail(NVFP4_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, L.total);

  AttnArgs a = {};
  a.B = batch->num_seqs;
  a.T = (int)batch->num_tokens;
  a.Hq = desc->num_heads;
  a.Hkv = desc->num_kv_heads;
  a.G = a.Hq / a.Hkv;
  a.D = desc->head_dim;
  a.page_size = cache->page_size;
  for (a.page_shift = 4; (1 << a.page_shift) < cache->page_size;) ++a.page_shift;
  a.max_pages = batch->max_pages;
  a.pt_stride = batch->page_table_stride;
  a.q_start = batch->q_start;
  a.kv_len = batch->kv_len;
  a.page_table = batch->page_table;
  a.visible = batch->visible_len;
  a.prefix_len = batch->prefix_len;
  a.causal = desc->causal != 0;
  // Positions stay below 2^30 (check_attention_batch), so a longer window masks
  // nothing either; below the first key, a position less a longer one would wrap.
  a.window = desc->window < 1 << 30 ? desc->window : 1 << 30;
  a.scale = desc->scale;
  a.softcap = desc->softcap;
  a.inv_cap = desc->softcap > 0.0f ? fminf(1.0f / desc->softcap, FLT_MAX) : 0.0f;  // (of a cap that is not normal)
  a.slopes = slopes;
  a.q = static_cast<const __nv_bfloat16 *>(q->data);
  a.q_ts = q->token_stride;
  a.q_hs = q->head_stride;
  a.gate = gate ? static_cast<const __nv_bfloat16 *>(gate->data) : nullptr;
  a.g_ts = gate ? gate->token_stride : 0;
  a.g_hs = gate ? gate->head_stride : 0;
  a.out = static_cast<__nv_bfloat16 *>(out->data);
  a.o_ts = out->token_stride;
  a.o_hs = out->head_stride;
  a.lse = lse;
  uint8_t *w = static_cast<uint8_t *>(ws);
  a.part_o = reinterpret_cast<float *>(w + L.part_o);
  a.part_ml = reinterpret_cast<float2 *>(w + L.part_ml);
  a.meta = reinterpret_cast<AttnMeta *>(w + L.meta);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pass = [&](int R, int64_t rows, const char *what) -> int {
    a.max_rows = (int)(rows < 1 << 30 ? rows : 1 << 30);
    a.max_blocks = (a.max_rows + R - 1) / R;
    // A box of the cache map: a page, or as much of it as a key tile takes.
    const int tile = R <= 32 ? attn_rows_tile(desc->head_dim) : 64;
    const int box = cache->page_size < tile ? cache->page_size : tile;
    // One copy for all columns where they fill the kernel's tile; the MMA on keys
    // also needs the tile's rows in one piece.
    a.wide_v = desc->head_dim == L.dp;
    a.wide = a.wide_v && (R <= 32 || box == tile);
    CUtensorMap tk, tv;
    if (!make_cache_map(&tk, cache->k, cache->k_strides, *cache, box, a.wide) ||
        !make_cache_map(&tv, cache->v, cache->v_strides, *cache, box, a.wide_v))
      return fail(NVFP4_ERR_CUDA, "tensor map of the cache");
    return check_launch(R <= 32 ? launch_attn_rows(tk, tv, a, R, grid, st) : launch_attn_tc(tk, tv, a, grid, st),
                        what);
  };
  if (batch->prefix_len > 0) {
    // All tokens against the shared prefix first: its keys are read once for
    // the whole batch; the own pass joins the result in its last step.
    a.prev_o = reinterpret_cast<float *>(w + L.prev_o);
    a.prev_lse = reinterpret_cast<float *>(w + L.prev_lse);
    a.prefix_pass = 1;
    a.page_table = batch->prefix_pages;
    if ((rc = pass(L.R0, (int64_t)a.T * a.G, "attention launch (prefix)"))) return rc;
    a.prefix_pass = 0;
    a.page_table = batch->page_table;
  }
  return pass(L.R1, (int64_t)batch->max_q_len * a.G, "attention launch");
}
