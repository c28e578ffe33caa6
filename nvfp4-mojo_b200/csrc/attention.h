// attention.h -- internals shared by the attention translation units
// (include/nvfp4_attention.h).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/nvfp4_attention.h"
#include "abi_util.h"

namespace nvfp4 {

// Checks of the structs that both entry points take: NVFP4_OK, or an error
// with its message recorded.
int check_kv_cache(const nvfp4_kv_cache *c);
int check_attention_batch(const nvfp4_attention_batch *b, int page_size);

// Streaming multiprocessors of the current device.
int attn_sms();

// What a call reads or writes of `tokens` x `heads` rows of `dim` values.
inline RowSpan head_span(const nvfp4_head_rows &r, int64_t tokens, int64_t heads, int dim, int esize) {
  return RowSpan{r.data, (int64_t)dim * esize, {tokens, heads}, {r.token_stride * esize, r.head_stride * esize}};
}

}  // namespace nvfp4
