// norm.cu -- the norms around a block fused with its gate and residual
// (include/nvfp4_norm.h).
//
// One pass: a row's x, residual and gate are read once into registers, both
// sums of squares (of x for the norm after the block, of the new residual for
// the norm before the next one) are reduced over the row's threads in fp32,
// and the new residual and the normed row are written once.  Bound by HBM
// for many rows (16384 rows of 2048, norms on both sides, fp32 residual and a
// gate: 76 us, 5.3 of the 6.6 TB/s that a copy reaches) and by latency for a few
// (one row: 2.1 us, the loads and one block-wide sum per norm).
#include <cuda_bf16.h>

#include "../../include/nvfp4.h"
#include "../../include/nvfp4_norm.h"
#include "abi_util.h"
#include "kernels.h"

namespace nvfp4 {
namespace {

struct NormArgs {
  nvfp4_norm_desc d;
  const void *x, *residual;
  const __nv_bfloat16 *post, *gate, *pre;
  void *r_out, *y;
};

// 8 consecutive values of a row as fp32 (16-byte loads), or 8 values nt apart.
template <bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const void *base, int dtype, int64_t row_off,
                                      int col, int nt, int H) {
  if constexpr (VEC) {
    if (dtype == kBF16) {
      const uint4 q =
          *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(base) + row_off + col);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + row_off + col);
      const float4 a = p[0], b = p[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
      v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col + i * nt;
      v[i] = c >= H ? 0.0f
             : dtype == kBF16
                 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(base)[row_off + c])
                 : static_cast<const float *>(base)[row_off + c];
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(const float (&v)[8], void *base, int dtype, int64_t row_off,
                                       int col, int nt, int H) {
  if constexpr (VEC) {
    if (dtype == kBF16) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
      *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(base) + row_off + col) =
          make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(base) + row_off + col);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col + i * nt;
      if (c < H) {
        if (dtype == kBF16)
          static_cast<__nv_bfloat16 *>(base)[row_off + c] = __float2bfloat16(v[i]);
        else
          static_cast<float *>(base)[row_off + c] = v[i];
      }
    }
  }
}

// Sum over the nt threads of a row: a warp, or the whole block, whose warps
// meet in `red`.
__device__ __forceinline__ float row_sum(float s, int nt, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (nt > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.0f;
    for (int i = 0; i < (nt >> 5); ++i) s += red[i];
  }
  return s;
}

// nt threads per row (32: eight rows per block, else a block per row), VPT
// groups of 8 values per thread.
template <int VPT, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : 1280 / THREADS) norm_residual_kernel(NormArgs a, int nt) {
  __shared__ float red[2][32];  // one per sum: the second needs no barrier before it
  const nvfp4_norm_desc &d = a.d;
  const int H = d.hidden, t = nt == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = nt == 32 ? (int64_t)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
  const bool live = row < d.rows;
  const float inv_h = 1.0f / (float)H;
  asm volatile("griddepcontrol.launch_dependents;");

  asm volatile("griddepcontrol.wait;" ::: "memory");
  float u[VPT][8], r[VPT][8];
  int col[VPT];
  bool in[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    col[v] = VEC ? (v * nt + t) * 8 : v * nt * 8 + t;
    in[v] = live && col[v] < H;
#pragma unroll
    for (int i = 0; i < 8; ++i) u[v][i] = r[v][i] = 0.0f;
    if (in[v]) {
      load8<VEC>(u[v], a.x, d.x_dtype, row * d.x_stride, col[v], nt, H);
      if (a.residual) load8<VEC>(r[v], a.residual, d.residual_dtype, row * d.residual_stride, col[v], nt, H);
    }
  }
  if (a.post) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(u[v][i], u[v][i], s);
    const float inv = rsqrtf(row_sum(s, nt, red[0]) * inv_h + d.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (in[v]) {
        float w[8];
        load8<VEC>(w, a.post, kBF16, 0, col[v], nt, H);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] *= inv * (w[i] + d.weight_offset);
      }
  }
  const bool sig = d.gate_act == NVFP4_GATE_SIGMOID;
  float row_gate = d.residual_scale;
  if (a.gate && d.gate_col_stride == 0 && live) {
    const float g = __bfloat162float(a.gate[row * d.gate_row_stride]);
    row_gate *= sig ? 1.0f / (1.0f + __expf(-g)) : g;
  }
  float s = 0.0f;
#pragma unroll
  for (int v = 0; v < VPT; ++v)
    if (in[v]) {
      if (a.gate && d.gate_col_stride) {
        float g[8];
        load8<VEC>(g, a.gate, kBF16, row * d.gate_row_stride, col[v], nt, H);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[v][i] *= sig ? 1.0f / (1.0f + __expf(-g[i])) : g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[v][i] = fmaf(row_gate, u[v][i], r[v][i]);
        if (VEC || col[v] + i * nt < H) s = fmaf(r[v][i], r[v][i], s);
      }
      if (a.r_out) store8<VEC>(r[v], a.r_out, d.residual_dtype, row * d.residual_out_stride, col[v], nt, H);
    }
  if (a.pre) {
    const float inv = rsqrtf(row_sum(s, nt, red[1]) * inv_h + d.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (in[v]) {
        float w[8];
        load8<VEC>(w, a.pre, kBF16, 0, col[v], nt, H);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[v][i] *= inv * (w[i] + d.weight_offset);
        store8<VEC>(r[v], a.y, d.y_dtype, row * d.y_stride, col[v], nt, H);
      }
  }
}

template <int VPT, bool VEC, int THREADS>
cudaError_t launch_norm_as(const NormArgs &a, int nt, cudaStream_t st) {
  const int rows_per_block = nt > 32 ? 1 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.d.rows + rows_per_block - 1) / rows_per_block), 1, 1);
  cfg.blockDim = dim3((unsigned)(nt * rows_per_block), 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_residual_kernel<VPT, VEC, THREADS>, a, nt);
}

template <int VPT, bool VEC>
cudaError_t launch_norm_vpt(const NormArgs &a, int nt, cudaStream_t st) {
  if constexpr (VPT < 4) {  // (four: rows beyond 16384)
    if (nt <= 32) return launch_norm_as<VPT, VEC, 256>(a, nt, st);
    if (nt <= 128) return launch_norm_as<VPT, VEC, 128>(a, nt, st);
    if (nt <= 256) return launch_norm_as<VPT, VEC, 256>(a, nt, st);
    if (nt <= 512) return launch_norm_as<VPT, VEC, 512>(a, nt, st);
  }
  return launch_norm_as<VPT, VEC, 1024>(a, nt, st);
}

template <bool VEC>
cudaError_t launch_norm(const NormArgs &a, cudaStream_t st) {
  // Few rows: 8 values a thread, for the shortest way through.  Rows enough to
  // fill the GPU: 16, so that more bytes are in flight per thread and fewer
  // threads meet at each sum (16384 rows of 2048, norms on both sides, fp32
  // residual: 86 us with 8 values a thread, 76 with 16, 96 with 32).  Rows of up
  // to 32 threads go eight to a block.
  const int H = a.d.hidden, per = H > 16384 ? 32 : H > 8192 || a.d.rows >= 592 ? 16 : 8;
  const int nt = ((H + per - 1) / per + 31) / 32 * 32;
  return per == 8 ? launch_norm_vpt<1, VEC>(a, nt, st)
         : per == 16 ? launch_norm_vpt<2, VEC>(a, nt, st)
                     : launch_norm_vpt<4, VEC>(a, nt, st);
}

bool norm_dt(int t) { return t == NVFP4_DTYPE_F32 || t == NVFP4_DTYPE_BF16; }

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_norm_residual(const nvfp4_norm_desc *d, const void *x, const void *residual,
                                   const void *post, const void *gate, const void *pre,
                                   void *r_out, void *y, void *stream) {
  NVFP4_ABI_RANGE();
  if (!d) return fail(NVFP4_ERR_INVALID_ARG, "null norm descriptor");
  if (d->rows < 0 || d->rows > INT32_MAX || d->hidden <= 0 || d->hidden > 32768)
    return fail(NVFP4_ERR_INVALID_ARG, "bad norm shape rows=%lld hidden=%d", (long long)d->rows, d->hidden);
  if (!norm_dt(d->x_dtype) || !norm_dt(d->residual_dtype) || !norm_dt(d->y_dtype))
    return fail(NVFP4_ERR_INVALID_ARG, "bad dtype");
  if (d->gate_act != NVFP4_GATE_LINEAR && d->gate_act != NVFP4_GATE_SIGMOID)
    return fail(NVFP4_ERR_INVALID_ARG, "bad gate activation %d", d->gate_act);
  if (!(d->eps >= 0.0f)) return fail(NVFP4_ERR_INVALID_ARG, "eps must not be negative");
  if (gate && d->gate_col_stride != 0 && d->gate_col_stride != 1)
    return fail(NVFP4_ERR_INVALID_ARG, "gate column stride must be 0 or 1");
  if (d->rows == 0) return NVFP4_OK;
  if (!r_out && !y) return fail(NVFP4_ERR_INVALID_ARG, "null residual_out and y: nothing to write");
  if ((y == nullptr) != (pre == nullptr))
    return fail(NVFP4_ERR_INVALID_ARG, "y and pre_weight go together: both or neither null");
  const int H = d->hidden;
  if (d->rows > 1 && (d->x_stride < H || (residual && d->residual_stride < H) ||
                      (r_out && d->residual_out_stride < H) || (y && d->y_stride < H)))
    return fail(NVFP4_ERR_INVALID_ARG, "row strides must be at least hidden");
  if (gate && d->gate_row_stride < 0) return fail(NVFP4_ERR_INVALID_ARG, "negative gate stride");
  // A row is read whole before it is written, by the same threads at the same
  // places: the outputs may be the inputs, but not shifted against them.
  if (r_out && r_out == residual && d->residual_out_stride != d->residual_stride)
    return fail(NVFP4_ERR_INVALID_ARG, "residual_out is residual with another stride");
  if (r_out && r_out == x && (d->residual_out_stride != d->x_stride || d->residual_dtype != d->x_dtype))
    return fail(NVFP4_ERR_INVALID_ARG, "residual_out is x with another stride or dtype");
  if (y && y == x && (d->y_stride != d->x_stride || d->y_dtype != d->x_dtype))
    return fail(NVFP4_ERR_INVALID_ARG, "y is x with another stride or dtype");
  if (y && y == residual && (d->y_stride != d->residual_stride || d->y_dtype != d->residual_dtype))
    return fail(NVFP4_ERR_INVALID_ARG, "y is residual with another stride or dtype");
  if (y && y == r_out) return fail(NVFP4_ERR_INVALID_ARG, "y and residual_out are the same buffer");
  if (!x) return fail(NVFP4_ERR_INVALID_ARG, "null x");
  auto span = [&](const void *p, int dt, int64_t stride, int64_t cols) {
    const int es = dt == kBF16 ? 2 : 4;
    return RowSpan{p, cols * es, {d->rows, 1}, {stride * es, 0}};
  };
  const RowSpan outs[2] = {span(r_out, d->residual_dtype, d->residual_out_stride, H), span(y, d->y_dtype, d->y_stride, H)};
  const RowSpan ins[3] = {span(x, d->x_dtype, d->x_stride, H), span(residual, d->residual_dtype, d->residual_stride, H),
                          span(gate, kBF16, d->gate_row_stride, d->gate_col_stride ? H : 1)};
  for (const RowSpan &o : outs)
    for (const RowSpan &i : ins)
      if (o.base && i.base && !same_rows(o, i) && rows_overlap(o, i))
        return fail(NVFP4_ERR_INVALID_ARG, "an output overlaps x, residual or gate in other places than its own");
  if (r_out && y && rows_overlap(outs[0], outs[1])) return fail(NVFP4_ERR_INVALID_ARG, "y and residual_out overlap");
  NormArgs a;
  a.d = *d;
  a.x = x;
  a.residual = residual;
  a.post = static_cast<const __nv_bfloat16 *>(post);
  a.gate = static_cast<const __nv_bfloat16 *>(gate);
  a.pre = static_cast<const __nv_bfloat16 *>(pre);
  a.r_out = r_out;
  a.y = y;
  // 16-byte accesses where every row starts on 16 bytes; otherwise by element.
  auto esize = [](int t) { return t == kBF16 ? 2 : 4; };
  auto fits = [&](const void *p, int dt, int64_t stride) {
    return !p || (aligned(p, 16) && (stride * esize(dt)) % 16 == 0);
  };
  const bool vec = H % 8 == 0 && fits(x, d->x_dtype, d->x_stride) &&
                   fits(residual, d->residual_dtype, d->residual_stride) &&
                   fits(r_out, d->residual_dtype, d->residual_out_stride) &&
                   fits(y, d->y_dtype, d->y_stride) && fits(post, kBF16, 0) && fits(pre, kBF16, 0) &&
                   (d->gate_col_stride == 0 || fits(gate, kBF16, d->gate_row_stride));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return check_launch(vec ? launch_norm<true>(a, st) : launch_norm<false>(a, st),
                      "norm launch");
}
