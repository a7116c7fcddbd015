// Shared device helpers of the sequence-model operators beside the loss (cross attention, head norm with
// rotation, gradient clipping): element types, per-sample lengths, vector loads.
#pragma once

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sdtw_b200.h"
#include "sdtw_common.cuh"

namespace sdtw {

// SMs of the current device, asked of the driver once (a decoded token's call is bound by the host).
inline cudaError_t current_sms(int& dev, int& sms)
{
    static std::atomic<int> known[128];
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 128) return cudaErrorInvalidDevice;
    sms = known[dev].load(std::memory_order_relaxed);
    if (sms > 0) return cudaSuccess;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) known[dev].store(sms, std::memory_order_relaxed);
    return e;
}

// Allows a kernel its dynamic shared memory, once a device (`done`: one flag a device, of this kernel alone).
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<bool> (&done)[128])
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 128) return cudaErrorInvalidDevice;
    if (done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_relaxed);
    return e;
}

inline size_t dtype_size(int dt) { return dt == SDTW_F64 ? 8 : (dt == SDTW_F32 ? 4 : 2); }

// A lengths array (null: every sample is full). get() returns the length of sample b out of `full`, or -1
// when it lies outside [0, full]; the kernels then treat the sample as bad and report it.
struct Lens {
    const void* p;
    int is32;
    __device__ __forceinline__ int64_t get(int64_t b, int64_t full) const
    {
        if (p == nullptr) return full;
        const int64_t n =
            is32 ? static_cast<int64_t>(static_cast<const int*>(p)[b]) : static_cast<const int64_t*>(p)[b];
        return n < 0 || n > full ? -1 : n;
    }
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x)
{
    return x;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x)
{
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x)
{
    return __float2bfloat16_rn(x);
}

// Two 16-bit numbers in a word.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// V elements moved as one access of V * sizeof(T) bytes (16 at most, aligned to that size).
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
    T e[V];
};

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
__device__ __forceinline__ float warp_maxf(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

}  // namespace sdtw
