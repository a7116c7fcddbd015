// Cross attention on warp-level mma: few query rows (states split over CTAs), float32, and any strides and alignment.
#pragma once

#include "sdtw_attention.h"

namespace sdtw {

size_t attention_split_workspace_bytes(const AttnArgs& a, int dtype);

// out, out_lo and lse of a (B, N > 0).
cudaError_t attention_split_forward(const AttnArgs& a, int dtype, void* workspace, cudaStream_t s);

// dq, dk, dv and delta of a (B > 0), fp16 behind attention_peaks.
cudaError_t attention_mma_backward(const AttnArgs& a, int dtype, cudaStream_t s);

}  // namespace sdtw
