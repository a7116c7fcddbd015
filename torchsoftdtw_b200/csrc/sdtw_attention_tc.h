// The tensor-core kernels of cross attention (16-bit operands).
#pragma once

#include <cuda.h>

#include "sdtw_attention.h"

namespace sdtw {

// Which kernel of the next calls has one warp withhold its first arrival (1 forward, 2 dq, 3 dk and dv; 0 none), so that the
// waits behind it run out: for tests of what happens then.
int attention_stall();

// Whether TMA can read the heads' tiles of this operand: 16-byte steps in every dimension.
bool attention_tc_takes(const void* p, const Strides& st, int64_t B, int64_t rows, int64_t H, int64_t d);

// Makes the current device's context the calling thread's, which the driver needs to encode a tensor map: a thread whose first
// CUDA call this is (autograd's, in a process whose first gradient is this one) has none yet.
cudaError_t attention_bind_context();

// TMA map of tiles of box_rows rows x 64 features of one head of (B, rows, H, d), 128-byte swizzle; what lies outside reads
// as zero.
bool attention_tile_map(CUtensorMap* map, bool half, const void* ptr, const Strides& st, int64_t B, int64_t rows, int64_t H,
                        int64_t d, int box_rows);

// out, out_lo and lse of a (M > 0), from q, k and v that attention_tc_takes.
cudaError_t attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s);

// dq, dk, dv and delta of a (N, M > 0), from q, k, v and dout that attention_tc_takes; fp16 behind
// attention_peaks.
cudaError_t attention_tc_backward(const AttnArgs& a, bool bf16, cudaStream_t s);

}  // namespace sdtw
