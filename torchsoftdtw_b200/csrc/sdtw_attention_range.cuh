// The scale of fp16 dS in the gradients of cross attention.
//
// dS_ij = P_ij (dP_ij - delta_i) goes through a product as a 16-bit operand. |dP_ij| <= |do_i| |v_j|, and delta_i, a mean of
// the row's dP, is known. So the largest |v| of the states that a tile of rows reaches bounds a row's dS, and the largest
// |do|, |delta| and |v| bound a state's; dS is scaled by a power of two that brings the bound to [2^14, 2^15), half of what
// fp16 holds, or below it by rounding. It never overflows, and what lies under fp16's normal numbers is 2^-28 of the bound and
// less (rounded by 2^-39 of it). With P kept 2^14 larger (2^-39 a cell) dq, dk and dv then lose bits to the type only where a
// |do| |v| that one CTA reaches is 2^24 and more below another. The maxima are kept over 64 rows: the values' from a pass over V
// (attention_peaks), do's and delta's from the dq kernels, through integer maxima, which have no order.
#pragma once

#include "sdtw_attention.h"

namespace sdtw {

constexpr float kHalfShift = 14.f;             // log2 of what fp16 P is kept larger by in the gradients
constexpr float kHalfUnshift = 0x1p-14f;

// A lane's part of the largest of p[first .. last] (numbers that are not negative). Joined over the warp where it is used, so
// that the loads run beside what comes between.
struct PeakPart {
    float m[2];
};
__device__ __forceinline__ PeakPart peak_part(const float* p, int64_t first, int64_t last)
{
    PeakPart r;
    int64_t i = first + (threadIdx.x & 31);
    r.m[0] = i <= last ? p[i] : 0.f;
    r.m[1] = i + 32 <= last ? p[i + 32] : 0.f;
    for (i += 64; i <= last; i += 32) r.m[0] = fmaxf(r.m[0], p[i]);
    return r;
}
// (As integers, whose order is that of the numbers: one instruction.)
__device__ __forceinline__ float peak_of(const PeakPart& p)
{
    return __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(fmaxf(p.m[0], p.m[1]))));
}
// Of the |v| of states [lo, hi) of key head (b, hk), hi > lo.
__device__ __forceinline__ PeakPart value_part(const AttnArgs& a, int64_t b, int64_t hk, int64_t lo, int64_t hi)
{
    return peak_part(a.v_peak + (b * a.Hkv + hk) * a.v_blocks, lo / kPeakRows, (hi - 1) / kPeakRows);
}
// The bound on |dP - delta| between queries [q0, q1) (of all query heads) and states [j0, j1) of key head (b, hk), neither empty.
__device__ __forceinline__ float gradient_bound(const AttnArgs& a, int64_t b, int64_t hk, int64_t q0, int64_t q1, int64_t j0,
                                                int64_t j1)
{
    const int64_t at = (b * a.Hkv + hk) * a.q_blocks;
    const PeakPart v = value_part(a, b, hk, j0, j1);
    const PeakPart norm2 = peak_part(a.do_peak + at, q0 / kPeakRows, (q1 - 1) / kPeakRows);
    const PeakPart delta = peak_part(a.delta_peak + at, q0 / kPeakRows, (q1 - 1) / kPeakRows);
    return fmaf(sqrtf(peak_of(norm2)), peak_of(v), peak_of(delta));
}
// Takes the largest |do|^2 and |delta| of some queries of one 64-row block into its maxima.
__device__ __forceinline__ void raise_gradient_peak(const AttnArgs& a, int64_t b, int64_t hk, int64_t i, float norm2, float delta)
{
    const int64_t at = (b * a.Hkv + hk) * a.q_blocks + i / kPeakRows;
    atomicMax(reinterpret_cast<int*>(a.do_peak) + at, __float_as_int(norm2));
    atomicMax(reinterpret_cast<int*>(a.delta_peak) + at, __float_as_int(delta));
}

__device__ __forceinline__ float half_scale(float bound)
{
    if (!(bound > 1e-30f) || !(bound < 1e30f)) return 1.f;
    return exp2f(14.f - floorf(log2f(bound)));
}

// Fills v_peak, and clears do_peak and delta_peak, of a (fp16).
cudaError_t attention_peaks(const AttnArgs& a, cudaStream_t s);

}  // namespace sdtw
