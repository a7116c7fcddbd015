// The problem of one cross-attention call as the kernels see it.
#pragma once

#include <type_traits>

#include "sdtw_sequence.cuh"

namespace sdtw {

constexpr int kPeakRows = 64;  // rows (states, or queries) that share one word of the maxima below

struct Strides {
    int64_t b, n, h;
};

struct AttnArgs {
    const void *q, *k, *v;
    Strides qs, ks, vs;
    int64_t N, M;
    int B, Hq, Hkv, d, group;  // group = Hq / Hkv
    Lens lx, ly;
    int64_t bw;
    float scale;       // scale of the scores
    float scale_log2;  // scale / ln 2: the softmax runs in powers of two
    uint32_t* err;
    void *out, *out_lo;  // (B, N, Hq, d); out_lo may be null
    float* lse;          // (B, Hq, N); the forward's may be null
    // backward
    const void *o, *o_lo;
    const void* dout;
    Strides gs;
    void *dq, *dk, *dv;
    float* delta;  // (B, Hq, N): sum_j p_ij dp_ij
    // fp16 (sdtw_attention_range.cuh): per key head, the largest |v| of each kPeakRows states; the largest |do|^2 and |delta| of
    // each kPeakRows queries of its query heads
    float *v_peak, *do_peak, *delta_peak;
    int64_t v_blocks, q_blocks;
};

// What out_lo holds of an output's remainder (what rounding it to its type dropped): fp16's is kept 2^11 larger, about as large
// as the output itself, for the remainders of outputs below 2^-3 end among fp16's subnormal numbers.
template <typename T>
constexpr float kLoScale = std::is_same<T, __half>::value ? 0x1p11f : 1.f;

// The lengths of sample b, and whether one of them is out of range (reported; the sample is then empty).
__device__ __forceinline__ bool pair_lengths(const AttnArgs& a, int64_t b, int64_t& nx, int64_t& ny)
{
    nx = a.lx.get(b, a.N);
    ny = a.ly.get(b, a.M);
    if (nx >= 0 && ny >= 0) return true;
    nx = ny = 0;
    return false;
}

// [lo, hi): the columns of row i < nx.
__device__ __forceinline__ void row_cells(const AttnArgs& a, int64_t i, int64_t nx, int64_t ny, int64_t& lo,
                                          int64_t& hi)
{
    band_row_range(i, nx, ny, a.bw, lo, hi);
    hi += 1;
}

// [lo, hi): the rows whose cells include column j < ny (the band is symmetric in its two axes).
__device__ __forceinline__ void column_cells(const AttnArgs& a, int64_t j, int64_t nx, int64_t ny, int64_t& lo,
                                             int64_t& hi)
{
    band_row_range(j, ny, nx, a.bw, lo, hi);
    hi += 1;
}

}  // namespace sdtw
