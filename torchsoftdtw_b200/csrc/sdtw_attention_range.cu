// The largest |v| of every 64 states of a key head, ahead of fp16 gradients of cross attention (sdtw_attention_range.cuh), one CTA
// each, all of its loads in flight at once. Reads V once; with it a step of 4 x 4096 x 3001 x 8/2 x 128, band 256, ragged, takes 195 us
// where the scale from |do| alone took 187.
#include "sdtw_attention_range.cuh"

namespace sdtw {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRowsAWarp = kPeakRows / kWarps;

// VEC: rows start on 16 bytes and hold a multiple of 8 features, LPR lanes take one; else the 32 lanes of a warp do.
template <bool VEC, int LPR>
__global__ void __launch_bounds__(kThreads) attend_peaks_kernel(const __grid_constant__ AttnArgs a, int64_t blocks, int64_t words)
{
    __shared__ float tops[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; w < words;
         w += static_cast<int64_t>(gridDim.x) * kThreads)
        a.do_peak[w] = a.delta_peak[w] = 0.f;
    const int64_t id = blockIdx.x;
    if (id >= blocks) return;
    const int64_t head = id / a.v_blocks, j0 = id % a.v_blocks * kPeakRows + warp * kRowsAWarp, b = head / a.Hkv;
    int64_t nx, ny;
    pair_lengths(a, b, nx, ny);
    const __half* v = static_cast<const __half*>(a.v) + b * a.vs.b + head % a.Hkv * a.vs.h + j0 * a.vs.n;
    float top = 0.f;
    if constexpr (VEC) {
        constexpr int RPW = 32 / LPR, ROUNDS = kRowsAWarp / RPW;
        const int c = lane % LPR * 8;
        Vec<__half, 8> x[ROUNDS];
#pragma unroll
        for (int t = 0; t < ROUNDS; ++t) {
            const int r = t * RPW + lane / LPR;
            x[t] = Vec<__half, 8>{};
            if (j0 + r < ny && c < a.d) x[t] = *reinterpret_cast<const Vec<__half, 8>*>(v + r * a.vs.n + c);
        }
#pragma unroll
        for (int t = 0; t < ROUNDS; ++t) {
            float n2 = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) n2 = fmaf(to_f(x[t].e[e]), to_f(x[t].e[e]), n2);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) n2 += __shfl_xor_sync(kFull, n2, o);
            top = fmaxf(top, n2);
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < kRowsAWarp; ++r) {
            float n2 = 0.f;
            if (j0 + r < ny)
                for (int c = lane; c < a.d; c += 32) {
                    const float x = to_f(v[r * a.vs.n + c]);
                    n2 = fmaf(x, x, n2);
                }
            top = fmaxf(top, warp_sum(n2));
        }
    }
    top = warp_maxf(top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    if (threadIdx.x == 0) a.v_peak[id] = sqrtf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
}

}  // namespace

cudaError_t attention_peaks(const AttnArgs& a, cudaStream_t s)
{
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv, blocks = heads * a.v_blocks, words = heads * a.q_blocks;
    const unsigned grid = static_cast<unsigned>(blocks > 1 ? blocks : 1);
    const auto steps = [](int64_t stride, int64_t size) { return size == 1 || stride % 8 == 0; };
    const bool vec = a.d % 8 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0 && steps(a.vs.n, a.M) && steps(a.vs.h, a.Hkv) &&
                     steps(a.vs.b, a.B);
    if (vec && a.d <= 64)
        attend_peaks_kernel<true, 8><<<grid, kThreads, 0, s>>>(a, blocks, words);
    else if (vec)
        attend_peaks_kernel<true, 16><<<grid, kThreads, 0, s>>>(a, blocks, words);
    else
        attend_peaks_kernel<false, 1><<<grid, kThreads, 0, s>>>(a, blocks, words);
    count_launch();
    return cudaGetLastError();
}

}  // namespace sdtw
