// Cross attention of one series' queries to another series' states, and its gradients:
//   s_ij = scale q_i.k_j,  p_i = softmax_j s_ij over the row's cells,  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  dp_ij = do_i.v_j,  delta_i = sum_j p_ij dp_ij = do_i.o_i,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// The cells of a row are one interval of columns (lengths and band), so every mask is two comparisons. This file checks the
// C entry points' arguments and chooses the kernels.
#include <cmath>

#include "sdtw_attention_range.cuh"
#include "sdtw_attention_split.h"
#include "sdtw_attention_tc.h"

namespace sdtw {
namespace {

constexpr int kDMax = 128;
constexpr int64_t kMost = 1 << 24;  // rows of a sample, and samples

sdtw_status checked(const sdtw_attention_problem* p)
{
    if (p == nullptr) return SDTW_EINVAL;
    if (p->dtype != SDTW_F32 && p->dtype != SDTW_F16 && p->dtype != SDTW_BF16) return SDTW_EDTYPE;
    if (p->B < 0 || p->N < 0 || p->M < 0 || p->Hq < 1 || p->Hkv < 1 || p->Hq % p->Hkv != 0) return SDTW_EINVAL;
    if (p->B > kMost || p->N > kMost || p->M > kMost || p->Hq > 65535 || p->d < 1 || p->d > kDMax) return SDTW_EINVAL;
    if (static_cast<double>(p->B) * static_cast<double>(p->Hq) * static_cast<double>(p->N + p->M + 256) > 2e9)
        return SDTW_EINVAL;  // the rows of all heads are counted in 32 bits
    if (!std::isfinite(p->scale)) return SDTW_EINVAL;
    const bool rows = p->B > 0 && p->N > 0, states = p->B > 0 && p->M > 0;
    if ((rows && p->q == nullptr) || (states && (p->k == nullptr || p->v == nullptr))) return SDTW_EINVAL;
    if ((rows || states) && p->err_word == nullptr) return SDTW_EINVAL;
    return SDTW_OK;
}

int64_t peak_blocks(int64_t rows) { return (rows + kPeakRows - 1) / kPeakRows; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

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
    // A band as wide as the longer series holds every cell; wider ones would only overflow its products.
    a.bw = p->bandwidth < kMost ? p->bandwidth : kMost;
    a.scale = static_cast<float>(p->scale);
    a.scale_log2 = static_cast<float>(p->scale * 1.4426950408889634);
    a.err = p->err_word;
    return a;
}

bool takes_tc(const sdtw_attention_problem* p, const AttnArgs& a)
{
    return p->dtype != SDTW_F32 && p->M > 0 && attention_tc_takes(a.q, a.qs, a.B, a.N, a.Hq, a.d) &&
           attention_tc_takes(a.k, a.ks, a.B, a.M, a.Hkv, a.d) && attention_tc_takes(a.v, a.vs, a.B, a.M, a.Hkv, a.d);
}
// Whether the forward runs on the tcgen05 kernel. Up to 16 packed rows a key head read the cache at its bandwidth in the kernel
// that splits the states, whatever the batch. Above, that kernel takes about 2.6 us (d <= 64; 3.7 us above) a 64-row block
// and 64 states on each of two places an SM, beside 18 us; the tcgen05 kernel 0.85 us a 64-state step and wave of CTAs (128 rows,
// two CTAs an SM; d > 64: 256 rows, one), beside 5 us. Both measured in bf16 at 8 heads, 512 and 4096 states:
// N = 64, B = 1 and 64, M = 4096, d = 64: 24 and 269 us split, 52 and 132 us on tcgen05.
bool forward_tc(const sdtw_attention_problem* p, const AttnArgs& a)
{
    if (a.N * a.group <= 16 || !takes_tc(p, a)) return false;
    int dev = 0, sms = 0;
    if (current_sms(dev, sms) != cudaSuccess || sms <= 0) sms = 148;
    const bool wide = a.d > 64;
    const int64_t rows = wide ? 256 : 128, places = wide ? sms : 2 * sms, steps = (a.M + 63) / 64;
    const int64_t ctas = static_cast<int64_t>(a.B) * a.Hq * ((a.N + rows - 1) / rows), waves = (ctas + places - 1) / places;
    const int64_t blocks = static_cast<int64_t>(a.B) * a.Hkv * ((a.N * a.group + 63) / 64);
    const double tc = static_cast<double>(waves) * (0.85 * static_cast<double>(steps) + 5.0);
    const double split = 18.0 + (wide ? 3.7 : 2.6) * static_cast<double>(blocks) * static_cast<double>(steps) / (2.0 * sms);
    return tc < split;
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
    if (out == nullptr || !aligned16(out) || !aligned16(out_lo)) return SDTW_EINVAL;
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
    using namespace sdtw;
    if (checked(p) != SDTW_OK) return 0;
    size_t words = static_cast<size_t>(p->B) * p->Hq * p->N;  // delta
    if (p->dtype == SDTW_F16) words += static_cast<size_t>(p->B) * p->Hkv * (peak_blocks(p->M) + 2 * peak_blocks(p->N));
    return words * sizeof(float);
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
    if (!aligned16(out) || !aligned16(out_lo) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return SDTW_EINVAL;
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
    if (p->dtype == SDTW_F16) {
        const size_t heads = static_cast<size_t>(a.B) * a.Hkv;
        a.v_blocks = peak_blocks(a.M);
        a.q_blocks = peak_blocks(a.N);
        a.v_peak = a.delta + static_cast<size_t>(a.B) * a.Hq * a.N;
        a.do_peak = a.v_peak + heads * a.v_blocks;
        a.delta_peak = a.do_peak + heads * a.q_blocks;
        const cudaError_t e = attention_peaks(a, s);
        if (e != cudaSuccess) return static_cast<sdtw_status>(e);
    }
    if (p->N > 0 && takes_tc(p, a) && attention_tc_takes(a.dout, a.gs, a.B, a.N, a.Hq, a.d))
        return static_cast<sdtw_status>(attention_tc_backward(a, p->dtype == SDTW_BF16, s));
    return static_cast<sdtw_status>(attention_mma_backward(a, p->dtype, s));
}

}  // extern "C"
