// What the files of the PyTorch operator layer share (defined in torch_ops.cpp).
#pragma once

#include <ATen/ATen.h>
#include <cuda_runtime.h>

#include "sdtw_b200.h"

namespace sdtw_ops {

// The sticky device error word of like's device.
uint32_t* error_word(const at::Tensor& like);
// Raises when a C-ABI call returned an error.
void check_status(sdtw_status st, const char* what);
// With TORCHSOFTDTW_B200_SYNC_CHECK=1: synchronises and raises on a device-side error.
void maybe_sync_check(const at::Tensor& like, cudaStream_t stream);

}  // namespace sdtw_ops
