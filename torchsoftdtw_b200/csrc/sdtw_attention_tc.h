// The tensor-core kernels of cross attention (16-bit operands).
#pragma once

#include "sdtw_attention.h"

namespace sdtw {

// Whether TMA can read the heads' tiles of this operand: 16-byte steps in every dimension.
bool attention_tc_takes(const void* p, const Strides& st, int64_t B, int64_t rows, int64_t H, int64_t d);

// out, out_lo and lse of a (M > 0), from q, k and v that attention_tc_takes.
cudaError_t attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s);

}  // namespace sdtw
