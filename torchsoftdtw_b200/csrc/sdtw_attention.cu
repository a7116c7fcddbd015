// Cross attention of one series' queries to another series' states, and its gradients:
//   s_ij = scale q_i.k_j,  p_i = softmax_j s_ij over the row's cells,  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  dp_ij = do_i.v_j,  delta_i = sum_j p_ij dp_ij = do_i.o_i,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// The cells of a row are one interval of columns (lengths and band), so every mask is two comparisons.
#include <cmath>

#include "sdtw_attention_split.h"
#include "sdtw_attention_tc.h"

namespace sdtw {
namespace {

constexpr int kRowThreads = 128;  // four warps, a row each
constexpr int kDMax = 128;

// One warp a query row: delta, then dq.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) attend_dq_rows_kernel(AttnArgs a)
{
    __shared__ float qs[kRowThreads / 32][kDMax], gs[kRowThreads / 32][kDMax];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + warp;
    if (row >= static_cast<int64_t>(a.B) * a.Hq * a.N) return;
    const int64_t i = row % a.N, h = row / a.N % a.Hq, b = row / a.N / a.Hq;
    int64_t nx, ny, lo = 0, hi = 0;
    if (!pair_lengths(a, b, nx, ny) && lane == 0) atomicOr(a.err, kErrBadLength);
    if (i < nx && ny > 0) row_cells(a, i, nx, ny, lo, hi);
    const T* qr = static_cast<const T*>(a.q) + b * a.qs.b + i * a.qs.n + h * a.qs.h;
    const T* gr = static_cast<const T*>(a.dout) + b * a.gs.b + i * a.gs.n + h * a.gs.h;
    const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + h / a.group * a.ks.h;
    const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + h / a.group * a.vs.h;
    const int64_t at = ((b * a.N + i) * a.Hq + h) * a.d;
    float delta = 0.f;
    if (hi > lo)
        for (int f = lane; f < a.d; f += 32) {
            qs[warp][f] = to_f(qr[f]) * a.scale_log2;
            gs[warp][f] = to_f(gr[f]);
            float o = to_f(static_cast<const T*>(a.o)[at + f]);
            if (a.o_lo) o += to_f(static_cast<const T*>(a.o_lo)[at + f]);
            delta = fmaf(gs[warp][f], o, delta);
        }
    delta = warp_sum(delta);
    __syncwarp();
    const float lse = a.lse[(b * a.Hq + h) * a.N + i];
    if (lane == 0) a.delta[(b * a.Hq + h) * a.N + i] = delta;
    float dq[kDMax / 32] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j0 = lo; j0 < hi; j0 += 32) {
        const int64_t j = j0 + lane;
        float ds = 0.f;
        if (j < hi) {
            const T *kr = kb + j * a.ks.n, *vr = vb + j * a.vs.n;
            float s = 0.f, dp = 0.f;
            for (int f = 0; f < a.d; ++f) {
                s = fmaf(qs[warp][f], to_f(kr[f]), s);
                dp = fmaf(gs[warp][f], to_f(vr[f]), dp);
            }
            ds = exp2f(s - lse) * (dp - delta);
        }
        const int cells = static_cast<int>(hi - j0 < 32 ? hi - j0 : 32);
        for (int t = 0; t < cells; ++t) {
            const float dt = __shfl_sync(kFull, ds, t);
            const T* kr = kb + (j0 + t) * a.ks.n;
#pragma unroll
            for (int e = 0; e < kDMax / 32; ++e)
                if (lane + 32 * e < a.d) dq[e] = fmaf(dt, to_f(kr[lane + 32 * e]), dq[e]);
        }
    }
    T* out = static_cast<T*>(a.dq) + at;
#pragma unroll
    for (int e = 0; e < kDMax / 32; ++e)
        if (lane + 32 * e < a.d) out[lane + 32 * e] = from_f<T>(dq[e] * a.scale);
}

// One warp a state: its rows of every query head that shares the state's head, in order.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) attend_dkdv_rows_kernel(AttnArgs a)
{
    __shared__ float ks[kRowThreads / 32][kDMax], vs[kRowThreads / 32][kDMax];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + warp;
    if (row >= static_cast<int64_t>(a.B) * a.Hkv * a.M) return;
    const int64_t j = row % a.M, hk = row / a.M % a.Hkv, b = row / a.M / a.Hkv;
    int64_t nx, ny, lo = 0, hi = 0;
    pair_lengths(a, b, nx, ny);
    if (j < ny && nx > 0) column_cells(a, j, nx, ny, lo, hi);
    const T* kr = static_cast<const T*>(a.k) + b * a.ks.b + j * a.ks.n + hk * a.ks.h;
    const T* vr = static_cast<const T*>(a.v) + b * a.vs.b + j * a.vs.n + hk * a.vs.h;
    if (hi > lo)
        for (int f = lane; f < a.d; f += 32) {
            ks[warp][f] = to_f(kr[f]) * a.scale_log2;
            vs[warp][f] = to_f(vr[f]);
        }
    __syncwarp();
    float dk[kDMax / 32] = {0.f, 0.f, 0.f, 0.f}, dv[kDMax / 32] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t h = hk * a.group; h < (hk + 1) * a.group; ++h) {
        const T* qb = static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h;
        const T* gb = static_cast<const T*>(a.dout) + b * a.gs.b + h * a.gs.h;
        for (int64_t i0 = lo; i0 < hi; i0 += 32) {
            const int64_t i = i0 + lane;
            float p = 0.f, ds = 0.f;
            if (i < hi) {
                const T *qr = qb + i * a.qs.n, *gr = gb + i * a.gs.n;
                float s = 0.f, dp = 0.f;
                for (int f = 0; f < a.d; ++f) {
                    s = fmaf(to_f(qr[f]), ks[warp][f], s);
                    dp = fmaf(to_f(gr[f]), vs[warp][f], dp);
                }
                const int64_t at = (b * a.Hq + h) * a.N + i;
                p = exp2f(s - a.lse[at]);
                ds = p * (dp - a.delta[at]);
            }
            const int cells = static_cast<int>(hi - i0 < 32 ? hi - i0 : 32);
            for (int t = 0; t < cells; ++t) {
                const float pt = __shfl_sync(kFull, p, t), dt = __shfl_sync(kFull, ds, t);
                const T *qr = qb + (i0 + t) * a.qs.n, *gr = gb + (i0 + t) * a.gs.n;
#pragma unroll
                for (int e = 0; e < kDMax / 32; ++e)
                    if (lane + 32 * e < a.d) {
                        dv[e] = fmaf(pt, to_f(gr[lane + 32 * e]), dv[e]);
                        dk[e] = fmaf(dt, to_f(qr[lane + 32 * e]), dk[e]);
                    }
            }
        }
    }
    const int64_t at = ((b * a.M + j) * a.Hkv + hk) * a.d;
#pragma unroll
    for (int e = 0; e < kDMax / 32; ++e)
        if (lane + 32 * e < a.d) {
            static_cast<T*>(a.dk)[at + lane + 32 * e] = from_f<T>(dk[e] * a.scale);
            static_cast<T*>(a.dv)[at + lane + 32 * e] = from_f<T>(dv[e]);
        }
}

sdtw_status checked(const sdtw_attention_problem* p)
{
    if (p == nullptr) return SDTW_EINVAL;
    if (p->dtype != SDTW_F32 && p->dtype != SDTW_F16 && p->dtype != SDTW_BF16) return SDTW_EDTYPE;
    constexpr int64_t kMost = 1 << 24;  // rows of a sample, heads and samples are counted in 32 bits
    if (p->B < 0 || p->N < 0 || p->M < 0 || p->Hq < 1 || p->Hkv < 1 || p->Hq % p->Hkv != 0) return SDTW_EINVAL;
    if (p->B > kMost || p->N > kMost || p->M > kMost || p->Hq > 65535 || p->d < 1 || p->d > kDMax) return SDTW_EINVAL;
    if (static_cast<double>(p->B) * static_cast<double>(p->Hq) * static_cast<double>(p->N + p->M + 256) > 2e9)
        return SDTW_EINVAL;  // one warp a row: the rows of all heads fit a grid
    if (!std::isfinite(p->scale)) return SDTW_EINVAL;
    const bool rows = p->B > 0 && p->N > 0, states = p->B > 0 && p->M > 0;
    if ((rows && p->q == nullptr) || (states && (p->k == nullptr || p->v == nullptr))) return SDTW_EINVAL;
    if ((rows || states) && p->err_word == nullptr) return SDTW_EINVAL;
    return SDTW_OK;
}

AttnArgs args_of(const sdtw_attention_problem* p)
{
    AttnArgs a{};
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.qs = {p->q_stride[0], p->q_stride[1], p->q_stride[2]};
    a.ks = {p->k_stride[0], p->k_stride[1], p->k_stride[2]};
    a.vs = {p->v_stride[0], p->v_stride[1], p->v_stride[2]};
    a.N = p->N;
    a.M = p->M;
    a.B = static_cast<int>(p->B);
    a.Hq = static_cast<int>(p->Hq);
    a.Hkv = static_cast<int>(p->Hkv);
    a.d = static_cast<int>(p->d);
    a.group = a.Hq / a.Hkv;
    a.lx = {p->lengths_x, p->lengths_int32};
    a.ly = {p->lengths_y, p->lengths_int32};
    a.bw = p->bandwidth;
    a.scale = static_cast<float>(p->scale);
    a.scale_log2 = static_cast<float>(p->scale * 1.4426950408889634);
    a.err = p->err_word;
    return a;
}

unsigned row_ctas(int64_t rows) { return static_cast<unsigned>((rows + kRowThreads / 32 - 1) / (kRowThreads / 32)); }

template <typename T>
void backward_rows(const AttnArgs& a, cudaStream_t s)
{
    if (a.N > 0) {
        attend_dq_rows_kernel<T><<<row_ctas(static_cast<int64_t>(a.B) * a.Hq * a.N), kRowThreads, 0, s>>>(a);
        count_launch();
    }
    if (a.M > 0) {
        attend_dkdv_rows_kernel<T><<<row_ctas(static_cast<int64_t>(a.B) * a.Hkv * a.M), kRowThreads, 0, s>>>(a);
        count_launch();
    }
}

// The tensor-core kernels take 16-bit operands that TMA can read; below kSplitRows packed rows a key head the kernel that
// splits the states is faster.
constexpr int64_t kSplitRows = 64;

bool takes_tc(const sdtw_attention_problem* p, const AttnArgs& a)
{
    return p->dtype != SDTW_F32 && p->M > 0 && attention_tc_takes(a.q, a.qs, a.B, a.N, a.Hq, a.d) &&
           attention_tc_takes(a.k, a.ks, a.B, a.M, a.Hkv, a.d) && attention_tc_takes(a.v, a.vs, a.B, a.M, a.Hkv, a.d);
}
bool forward_tc(const sdtw_attention_problem* p, const AttnArgs& a)
{
    return a.N * a.group > kSplitRows && takes_tc(p, a);
}

sdtw_status last_error()
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SDTW_OK : static_cast<sdtw_status>(e);
}

}  // namespace
}  // namespace sdtw

extern "C" {

size_t sdtw_cross_attention_workspace_bytes(const sdtw_attention_problem* p)
{
    using namespace sdtw;
    if (checked(p) != SDTW_OK || p->B == 0 || p->N == 0) return 0;
    const AttnArgs a = args_of(p);
    return forward_tc(p, a) ? 0 : attention_split_workspace_bytes(a, p->dtype);
}

sdtw_status sdtw_cross_attention(const sdtw_attention_problem* p, void* out, void* out_lo, float* lse,
                                 void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace sdtw;
    const sdtw_status st = checked(p);
    if (st != SDTW_OK || p->B == 0 || p->N == 0) return st;
    if (out == nullptr || lse == nullptr) return SDTW_EINVAL;
    const size_t need = sdtw_cross_attention_workspace_bytes(p);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SDTW_EWORKSPACE;
    AttnArgs a = args_of(p);
    a.out = out;
    a.out_lo = out_lo;
    a.lse = lse;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (forward_tc(p, a)) return static_cast<sdtw_status>(attention_tc_forward(a, p->dtype == SDTW_BF16, s));
    return static_cast<sdtw_status>(attention_split_forward(a, p->dtype, workspace, s));
}

size_t sdtw_cross_attention_backward_workspace_bytes(const sdtw_attention_problem* p)
{
    if (sdtw::checked(p) != SDTW_OK) return 0;
    // delta, and a word a key head
    return (static_cast<size_t>(p->B) * p->Hq * p->N + static_cast<size_t>(p->B) * p->Hkv) * sizeof(float);
}

sdtw_status sdtw_cross_attention_backward(const sdtw_attention_problem* p, const void* out, const void* out_lo,
                                          const float* lse, const void* dout, const int64_t* dout_stride, void* dq,
                                          void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace sdtw;
    const sdtw_status st = checked(p);
    if (st != SDTW_OK || p->B == 0) return st;
    if (p->N > 0 && (out == nullptr || lse == nullptr || dout == nullptr || dout_stride == nullptr || dq == nullptr))
        return SDTW_EINVAL;
    if (p->M > 0 && (dk == nullptr || dv == nullptr)) return SDTW_EINVAL;
    const size_t need = sdtw_cross_attention_backward_workspace_bytes(p);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return SDTW_EWORKSPACE;
    AttnArgs a = args_of(p);
    a.o = out;
    a.o_lo = out_lo;
    a.lse = const_cast<float*>(lse);
    a.dout = dout;
    if (dout_stride) a.gs = {dout_stride[0], dout_stride[1], dout_stride[2]};
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.delta = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p->N > 0 && takes_tc(p, a) && attention_tc_takes(a.dout, a.gs, a.B, a.N, a.Hq, a.d)) {
        uint32_t* peak = reinterpret_cast<uint32_t*>(a.delta + static_cast<size_t>(a.B) * a.Hq * a.N);
        return static_cast<sdtw_status>(attention_tc_backward(a, p->dtype == SDTW_BF16, peak, s));
    }
    if (p->dtype == SDTW_F32)
        backward_rows<float>(a, s);
    else if (p->dtype == SDTW_F16)
        backward_rows<__half>(a, s);
    else
        backward_rows<__nv_bfloat16>(a, s);
    return last_error();
}

}  // extern "C"
