// attention_launch.h -- host launchers of the attention kernels.
#pragma once

#include <atomic>

#include "attention.cuh"

namespace nvfp4 {

// Lets a kernel use `bytes` of dynamic shared memory on the current device;
// `devices` remembers where that has been done.
cudaError_t attn_allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> &devices);

// attention_rows.cu: items of R = 16 or 32 rows (16 above head size 64), and
// the launch that joins what its workers (warps) cut.  Key tiles of
// attn_rows_tile tokens.
constexpr int kAttnRowsWorkers = 8;  // per block
inline int attn_rows_tile(int head_dim) { return head_dim <= 128 ? 32 : 16; }
cudaError_t launch_attn_rows(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int R,
                             int grid, cudaStream_t st);

// attention_tc.cu: items of 256 rows (128 above head size 128).
cudaError_t launch_attn_tc(const CUtensorMap &tk, const CUtensorMap &tv, const AttnArgs &a, int grid,
                           cudaStream_t st);

}  // namespace nvfp4
