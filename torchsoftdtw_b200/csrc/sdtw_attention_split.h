// Cross attention with the states split over CTAs: few query rows, and float32 (any strides, any alignment).
#pragma once

#include "sdtw_attention.h"

namespace sdtw {

size_t attention_split_workspace_bytes(const AttnArgs& a, int dtype);

// out, out_lo and lse of a (B, N > 0).
cudaError_t attention_split_forward(const AttnArgs& a, int dtype, void* workspace, cudaStream_t s);

}  // namespace sdtw
