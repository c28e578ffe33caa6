/*
 * nvfp4_norm.h -- the norms around a block fused with its gate and residual.
 * No reference counterpart as a function of its own (the reference norms each
 * head inside its DeltaNet step, nvfp4/deltanet.mojo:300-330).  Conventions
 * as in nvfp4.h.
 */
#ifndef NVFP4_NORM_H
#define NVFP4_NORM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum nvfp4_gate_act {
  NVFP4_GATE_LINEAR = 0,
  NVFP4_GATE_SIGMOID = 1,
} nvfp4_gate_act;

/*
 * Per row of `hidden` values:
 *   u = post_weight ? rms(x) * (post_weight + weight_offset) : x
 *   r = residual + residual_scale * act(gate) * u      (either may be missing)
 *   y = rms(r) * (pre_weight + weight_offset)
 * with rms(x) = x * rsqrt(mean x^2 + eps), in fp32; y is computed from r
 * before r is rounded.  x, residual and residual_out, and y have their own
 * dtypes (bf16 or f32); weights and gate are bf16.  Row strides in elements.
 */
typedef struct nvfp4_norm_desc {
  int64_t rows;
  int32_t hidden;                /* 1 .. 32768 */
  int32_t x_dtype;
  int32_t residual_dtype;
  int32_t y_dtype;
  int32_t gate_act;
  float residual_scale;
  float eps;
  float weight_offset;
  int64_t x_stride;
  int64_t residual_stride;
  int64_t residual_out_stride;
  int64_t y_stride;
  int64_t gate_row_stride;       /* 0: one gate row for all rows */
  int64_t gate_col_stride;       /* 1, or 0: one value per row */
} nvfp4_norm_desc;

/*
 * residual, post_weight and gate may be NULL; one of residual_out and y may
 * be NULL, and y is written where pre_weight is not NULL.  residual_out may
 * be residual or x (same dtype and stride); y may be x in the same way.  Other
 * overlaps of an output with x, residual, gate or the other output are refused.
 */
int nvfp4_norm_residual(const nvfp4_norm_desc *desc, const void *x, const void *residual,
                        const void *post_weight, const void *gate, const void *pre_weight,
                        void *residual_out, void *y, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NVFP4_NORM_H */
