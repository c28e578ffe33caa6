/*
 * nvfp4_attention.h -- softmax attention over a paged key/value cache, for
 * the attention layers of the models whose MoE and DeltaNet layers this
 * library runs: appending keys and values with the position rotation on the
 * way, and attention for prompts, for single tokens and for a batch that
 * shares a prefix.  No reference counterpart (the reference loads the
 * projections, nvfp4/weight_loader.mojo:776-893, and computes no attention).
 *
 * Conventions as in nvfp4.h: device pointers owned by the caller, 0 or a
 * negative nvfp4_status, work enqueued on `stream`.  Data is bf16 unless a
 * comment says otherwise; scores, softmax statistics, sums and partial results
 * are fp32.  The softmax's weights are rounded to bf16 for their product with
 * the values (the sum keeps them unrounded), which moves an output by at most
 * 2^-8 of the weighted mean of its |values|; exponentials and the gate's sigmoid
 * are within a few units of 2^-22.  Lengths, page tables and positions are int32 in device memory, so
 * that a captured graph can be replayed with new ones.  Device values that
 * contradict the descriptors are clamped, never followed out of range: a page
 * id outside [0, num_pages) reads as zeros and is not written, a length is
 * held to max_pages * page_size, a token range to [0, num_tokens].
 */
#ifndef NVFP4_ATTENTION_H
#define NVFP4_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of heads: element (token, head, d) at data + token * token_stride +
 * head * head_stride + d (strides in elements). */
typedef struct nvfp4_head_rows {
  void *data;
  int64_t token_stride;
  int64_t head_stride;
} nvfp4_head_rows;

/*
 * The cache: element (page, slot, head, d) of k at k + page * k_strides[0] +
 * slot * k_strides[1] + head * k_strides[2] + d, v the same.  Any order of
 * page, slot and head, and k and v interleaved in one buffer, are strides.
 * Pointers 16-byte aligned, strides multiples of 8 elements; page_size a
 * power of two in [16, 256]; head_dim a multiple of 8, at most 256.
 */
typedef struct nvfp4_kv_cache {
  void *k;
  void *v;
  int64_t k_strides[3];
  int64_t v_strides[3];
  int64_t num_pages;
  int32_t page_size;
  int32_t num_kv_heads;
  int32_t head_dim;
} nvfp4_kv_cache;

/*
 * One step's sequences.  Sequence b has the tokens q_start[b] ..
 * q_start[b + 1] - 1 of the call (q_start NULL: token b), which are the last
 * ones of its kv_len[b] keys; key j lies in page page_table[b *
 * page_table_stride + j / page_size], slot j % page_size.  With a shared
 * prefix, the prefix_len keys in prefix_pages come before every sequence's
 * own, which kv_len does not count.  A position below is that in the whole
 * sequence, prefix included.
 */
typedef struct nvfp4_attention_batch {
  int32_t num_seqs;
  int32_t max_q_len;            /* no sequence has more tokens in this call */
  int64_t num_tokens;
  const int32_t *q_start;       /* [num_seqs + 1], or NULL: num_seqs == num_tokens */
  const int32_t *kv_len;        /* [num_seqs], this call's tokens included */
  const int32_t *page_table;    /* [num_seqs, max_pages] */
  int64_t page_table_stride;    /* at least max_pages, or 0: one row for all sequences */
  int32_t max_pages;
  int32_t prefix_len;           /* 0: none */
  const int32_t *prefix_pages;  /* [ceil(prefix_len / page_size)] */
  const int32_t *visible_len;   /* [num_seqs] or NULL: the first visible_len[b]
                                   positions are seen by every query of b (that
                                   a window lets see so far back) */
} nvfp4_attention_batch;

/* Rotation of the first rotary_dim values of a head in pairs (i, i +
 * rotary_dim / 2), or (2 i, 2 i + 1) when interleaved, by the angle
 * position[axis[i]] * inv_freq[i]; both results times `scale`. */
typedef struct nvfp4_rotary {
  const float *inv_freq;        /* [rotary_dim / 2] */
  const int32_t *axis;          /* [rotary_dim / 2] or NULL: axis 0 */
  int32_t rotary_dim;           /* even, <= head_dim */
  int32_t interleaved;
  float scale;
} nvfp4_rotary;

/* RMS norm of each query / key head before the rotation: x * rsqrt(mean x^2 +
 * eps) * (weight + weight_offset), weights bf16 [head_dim], NULL: no norm. */
typedef struct nvfp4_qk_norm {
  const void *q_weight;
  const void *k_weight;
  float eps;
  float weight_offset;
} nvfp4_qk_norm;

/*
 * For every token of the batch: q normed and rotated into q_out (may be q
 * itself), k normed and rotated into the cache, v into the cache.  q, k, v
 * are rows of in_dtype (bf16 or f32), q_out and the cache bf16; other overlaps
 * of q_out's rows, with each other or with q, k and v, are refused.  positions
 * [num_axes, num_tokens] with row stride position_stride (0: one row for all
 * axes), or NULL: the token's position on every axis.  rotary or norm NULL: none.  The angle is
 * exact to fp32 for every int32 position.  A token whose key lies outside the
 * page table, or in a page outside the cache, gets its q_out but no key.  A
 * token outside every sequence leaves cache and q_out as they were.
 * Two tokens of one call must not share a key, and the cache's keys and values
 * must not share their places (the same pointer for both is refused).
 */
int nvfp4_kv_append(const nvfp4_kv_cache *cache, const nvfp4_attention_batch *batch,
                    const nvfp4_rotary *rotary, const nvfp4_qk_norm *norm,
                    const nvfp4_head_rows *q, const nvfp4_head_rows *k, const nvfp4_head_rows *v,
                    int in_dtype, int32_t num_heads, const int32_t *positions,
                    int64_t position_stride, int32_t num_axes, const nvfp4_head_rows *q_out,
                    void *stream);

/*
 * Attention of query position p over key positions j in [lo, hi):
 *   s = scale * q.k (scale > 0);  softcap > 0: s = softcap * tanh(s / softcap);
 *   slopes: s -= slopes[head] * |p - j|;
 *   hi = causal ? max(p + 1, visible_len) : all;  lo = window ? p - window + 1 : 0.
 * Query head h reads key/value head h / (num_heads / num_kv_heads); at most
 * 128 query heads to a key/value head.
 */
typedef struct nvfp4_attention_desc {
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t causal;
  int32_t window;
  float scale;
  float softcap;
} nvfp4_attention_desc;

/* Bytes of workspace that nvfp4_paged_attention needs on the current device
 * (0: the arguments are refused). */
size_t nvfp4_attention_workspace_size(const nvfp4_attention_desc *desc,
                                      const nvfp4_attention_batch *batch);

/*
 * out (token, head, :) = softmax(s) v, times sigmoid(gate) where gate is not
 * NULL; lse [num_tokens, num_heads] fp32 (may be NULL) the log-sum-exp of the
 * scores.  A query that sees no key gets 0 and -inf; a token outside every
 * sequence leaves out and lse as they were.  slopes fp32 [num_heads] or NULL.
 * q, out and gate 16-byte aligned with strides that are multiples of 8
 * elements; out may be q or gate (the same rows in the same places), and is
 * refused where its rows overlap theirs or each other otherwise.  The workspace (256-byte aligned, any contents) is
 * the call's own until it has finished: calls that may run at the same time
 * need one each.  Nothing beyond a sequence's keys is used, so what the rest
 * of its last page holds does not matter.  A key or value that is not finite
 * makes the outputs of the queries of the same call that read it, and may
 * make those of queries of the same sequence that do not, not finite.
 */
int nvfp4_paged_attention(const nvfp4_attention_desc *desc, const nvfp4_head_rows *q,
                          const nvfp4_kv_cache *cache, const nvfp4_attention_batch *batch,
                          const float *slopes, const nvfp4_head_rows *gate,
                          const nvfp4_head_rows *out, float *lse, void *workspace,
                          size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NVFP4_ATTENTION_H */
