// abi_util.h -- error reporting helpers shared by the C-ABI translation units.
#pragma once

#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>
#include <stddef.h>
#include <stdint.h>

namespace nvfp4 {

// Records a printf-style message as the thread's last error; returns `code`.
int fail(int code, const char *fmt, ...);
// NVFP4_OK, or NVFP4_ERR_CUDA with the CUDA error text recorded.
int check_launch(cudaError_t e, const char *what);
bool aligned(const void *p, size_t a);

// Rows of `bytes` bytes at base + i * stride[0] + j * stride[1], i < n[0] and
// j < n[1] (strides in bytes), for what a call reads or writes.
struct RowSpan {
  const void *base;
  int64_t bytes;
  int64_t n[2];
  int64_t stride[2];
};
// Two rows of one span share memory.
bool rows_overlap(const RowSpan &a);
// A row of a shares memory with one of b.  Exact for rows at the same strides
// (slices of one buffer) and for spans that lie apart; otherwise it may say so
// where the rows pass each other by.
bool rows_overlap(const RowSpan &a, const RowSpan &b);
// The same rows, each at its own place.
bool same_rows(const RowSpan &a, const RowSpan &b);

// An NVTX range named after the C-ABI call it wraps, so that Nsight tools
// (ncu --nvtx, nsys) attribute the kernels to the entry point that launched
// them.  Header-only NVTX: without a tool attached each push/pop is a few
// nanoseconds and nothing is loaded.
struct AbiRange {
  explicit AbiRange(const char *name) { nvtxRangePushA(name); }
  ~AbiRange() { nvtxRangePop(); }
  AbiRange(const AbiRange &) = delete;
  AbiRange &operator=(const AbiRange &) = delete;
};
#define NVFP4_ABI_RANGE() ::nvfp4::AbiRange nvfp4_abi_range_(__func__)

}  // namespace nvfp4
