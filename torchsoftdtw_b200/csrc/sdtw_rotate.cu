// RMS norm of every head followed by the rotation of its features by the position, and the gradient:
//   r = (mean(x^2) + eps)^(-1/2),  u = x r,  z = u w,  y = R z
//   R turns the pair p = 0 .. rotary/2 - 1 of z by the angle pos * base^(-2p / rotary); pairs are the features
//   (p, p + rotary/2), or (2p, 2p + 1) when interleaved; the features from `rotary` on stay.
//   backward: g = R^T dy, dw = sum g u, dx = r (g w - u mean(g w u)); r is formed again from x.
//
// Bound by memory: x in and y out; x and dy in, dx out. A head (d features) belongs to a group of G lanes, a
// lane to V neighbouring pairs (two vectors of V features), so the mean is log2 G shuffles and a pair never
// leaves its lane. A group takes one token and walks `hpu` of its heads: the angles (64-bit products, so that
// far positions keep theirs; then one sincospi a pair) are formed once for them. dw: every lane adds the products of its
// own features over all its tokens in 32 bits, the CTA joins its groups, a second launch joins the CTAs, each
// in a fixed order.
#include <cmath>
#include <mutex>

#include "sdtw_sequence.cuh"

namespace sdtw {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // d <= 256
constexpr int kCtasPerSm = 4;
constexpr int kMaxGradCtas = 1024;

struct RotArgs {
    const void* x;
    int64_t sb, sn, sh;  // strides of x in elements; features are neighbours
    const void* dy;      // backward
    int64_t gb, gn, gh;
    void* y;             // (B, N, H, d) contiguous: y, or dx
    const void* weight;  // null: ones
    int weight_f32;      // weight's type: float32, else x's
    const void* positions;  // null: the row index
    int pos_kind;        // 0 float32, 1 int32, 2 int64
    int64_t pb, pn;      // strides of the positions
    Lens len;
    uint32_t* err;
    int64_t tokens, N;
    int H, d, rotary, interleaved;
    int hpu, units_per_token;  // heads per unit of work
    float eps;
    float* dw;           // (grid, d) partial sums
    double turns[kMaxPairs];  // turns per position of pair p: base^(-2p / rotary) / (2 pi)
};

__device__ __forceinline__ double position(const RotArgs& a, int64_t b, int64_t n)
{
    if (a.positions == nullptr) return static_cast<double>(n);
    const int64_t at = b * a.pb + n * a.pn;
    if (a.pos_kind == 0) return static_cast<double>(static_cast<const float*>(a.positions)[at]);
    if (a.pos_kind == 1) return static_cast<double>(static_cast<const int*>(a.positions)[at]);
    return static_cast<double>(static_cast<const int64_t*>(a.positions)[at]);
}

template <int G>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Features of pair group `pg` (V pairs from p0 = pg V): the offsets of its two vectors, and whether it turns.
// The host only chooses V > 1 when V divides rotary / 2 and 2 V divides d, so a group is all of one kind.
template <int V>
__device__ __forceinline__ void pair_offsets(const RotArgs& a, int pg, int& oa, int& ob, bool& turned)
{
    const int p0 = pg * V, half = a.rotary / 2;
    turned = p0 < half;
    if (turned && !a.interleaved) {
        oa = p0;
        ob = p0 + half;
    } else {
        oa = 2 * p0;
        ob = 2 * p0 + V;
    }
}

// The 2V features of a lane: both vectors, the second from V on.
template <typename T, int V>
__device__ __forceinline__ void load_pairs(const T* row, int oa, int ob, int d, float (&f)[2 * V])
{
    if constexpr (V == 1) {
        f[0] = oa < d ? to_f(row[oa]) : 0.f;
        f[1] = ob < d ? to_f(row[ob]) : 0.f;
    } else {
        const Vec<T, V> va = *reinterpret_cast<const Vec<T, V>*>(row + oa);
        const Vec<T, V> vb = *reinterpret_cast<const Vec<T, V>*>(row + ob);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            f[i] = to_f(va.e[i]);
            f[V + i] = to_f(vb.e[i]);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_pairs(T* row, int oa, int ob, int d, const float (&f)[2 * V])
{
    if constexpr (V == 1) {
        if (oa < d) row[oa] = from_f<T>(f[0]);
        if (ob < d) row[ob] = from_f<T>(f[1]);
    } else {
        Vec<T, V> va, vb;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            va.e[i] = from_f<T>(f[i]);
            vb.e[i] = from_f<T>(f[V + i]);
        }
        *reinterpret_cast<Vec<T, V>*>(row + oa) = va;
        *reinterpret_cast<Vec<T, V>*>(row + ob) = vb;
    }
}

// Turn the V pairs by (c, s); sign -1 turns back.
template <int V>
__device__ __forceinline__ void turn(float (&f)[2 * V], const float (&c)[V], const float (&s)[V], bool split,
                                     float sign)
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float sn = sign * s[i];
        if (split) {
            const float p = f[i], q = f[V + i];
            f[i] = p * c[i] - q * sn;
            f[V + i] = p * sn + q * c[i];
        } else {
            const float p = f[2 * i], q = f[2 * i + 1];
            f[2 * i] = p * c[i] - q * sn;
            f[2 * i + 1] = p * sn + q * c[i];
        }
    }
}

// K pair groups a lane (1, or 4 with V = 1 and G = 32: any d up to 256, odd or unaligned).
template <typename T, int V, int G, int K, bool GRAD>
__global__ void __launch_bounds__(kThreads) norm_rotate_kernel(const __grid_constant__ RotArgs a)
{
    constexpr int kGroups = kThreads / G;
    __shared__ float red[GRAD ? kGroups * G * K * 2 * V : 1];
    const int gl = threadIdx.x % G, group = threadIdx.x / G;
    const int pair_groups = (a.d + 2 * V - 1) / (2 * V);
    int oa[K], ob[K];
    bool turned[K], live[K];
    float w[K][2 * V], dw[K][2 * V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int pg = gl + k * G;
        live[k] = pg < pair_groups;
        pair_offsets<V>(a, live[k] ? pg : 0, oa[k], ob[k], turned[k]);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
            const int o = i < V ? oa[k] + i : ob[k] + i - V;
            dw[k][i] = 0.f;
            w[k][i] = 1.f;
            if (a.weight != nullptr && live[k] && o < a.d)
                w[k][i] = a.weight_f32 ? static_cast<const float*>(a.weight)[o] : to_f(static_cast<const T*>(a.weight)[o]);
        }
    }
    const float inv_d = 1.f / static_cast<float>(a.d);
    const bool split = !a.interleaved;
    const int64_t units = a.tokens * a.units_per_token;
    // Every lane of a warp makes the same number of rounds (the shuffles need them all).
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kGroups;
    for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * kGroups; u0 < units; u0 += stride) {
        const int64_t u = u0 + group;
        const bool on = u < units;
        const int64_t token = on ? u / a.units_per_token : 0;
        const int h0 = on ? static_cast<int>(u - token * a.units_per_token) * a.hpu : 0;
        const int64_t b = token / a.N, n = token - b * a.N;
        const int64_t len = a.len.get(b, a.N);
        if (on && len < 0 && gl == 0) atomicOr(a.err, kErrBadLength);
        const bool valid = on && n < len;
        float c[K][V], s[K][V];
        const double pos = valid ? position(a, b, n) : 0.0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                c[k][i] = 1.f;
                s[k][i] = 0.f;
                if (live[k] && turned[k]) {
                    const double t = pos * a.turns[(gl + k * G) * V + i];
                    const float f = static_cast<float>(t - rint(t));  // turns beyond whole ones, in [-1/2, 1/2]
                    sincospif(2.f * f, &s[k][i], &c[k][i]);
                }
            }
        const float fill = on && len < 0 && !GRAD ? __int_as_float(0x7fc00000) : 0.f;
        for (int hh = 0; hh < a.hpu; ++hh) {
            const int h = h0 + hh;
            const bool head = on && h < a.H, work = valid && h < a.H;
            float f[K][2 * V], g[K][2 * V];
            float ss = 0.f, dot = 0.f;
            const T* xr = static_cast<const T*>(a.x) + b * a.sb + n * a.sn + h * a.sh;
            const T* gr = GRAD ? static_cast<const T*>(a.dy) + b * a.gb + n * a.gn + h * a.gh : nullptr;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) f[k][i] = g[k][i] = 0.f;
                if (work && live[k]) {
                    load_pairs<T, V>(xr, oa[k], ob[k], a.d, f[k]);
                    if constexpr (GRAD) load_pairs<T, V>(gr, oa[k], ob[k], a.d, g[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if constexpr (GRAD) {
                    if (turned[k]) turn<V>(g[k], c[k], s[k], split, -1.f);
                }
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    ss = fmaf(f[k][i], f[k][i], ss);
                    if constexpr (GRAD) dot = fmaf(g[k][i] * w[k][i], f[k][i], dot);
                }
            }
            ss = group_sum<G>(ss);
            if constexpr (GRAD) dot = group_sum<G>(dot);
            const float r = rsqrtf(ss * inv_d + a.eps);
            const float back = GRAD ? dot * inv_d * r * r : 0.f;
            T* yr = static_cast<T*>(a.y) + (token * a.H + h) * a.d;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if constexpr (GRAD) {
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) {
                        if (work) dw[k][i] = fmaf(g[k][i], f[k][i] * r, dw[k][i]);
                        g[k][i] = work ? r * (g[k][i] * w[k][i] - f[k][i] * back) : 0.f;
                    }
                    if (head && live[k]) store_pairs<T, V>(yr, oa[k], ob[k], a.d, g[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) f[k][i] = work ? f[k][i] * r * w[k][i] : fill;
                    if (work && turned[k]) turn<V>(f[k], c[k], s[k], split, 1.f);
                    if (head && live[k]) store_pairs<T, V>(yr, oa[k], ob[k], a.d, f[k]);
                }
            }
        }
    }
    if constexpr (GRAD) {
        if (a.dw == nullptr) return;
        // red[group][lane][k][i]; then the features' sums over the groups, in order.
        float* mine = red + (group * G + gl) * (K * 2 * V);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) mine[k * 2 * V + i] = dw[k][i];
        __syncthreads();
        for (int e = threadIdx.x; e < G * K * 2 * V; e += kThreads) {
            const int lane = e / (K * 2 * V), k = (e / (2 * V)) % K, i = e % (2 * V);
            const int pg = lane + k * G;
            if (pg >= pair_groups) continue;
            int fa, fb;
            bool tn;
            pair_offsets<V>(a, pg, fa, fb, tn);
            const int o = i < V ? fa + i : fb + i - V;
            if (o >= a.d) continue;
            float t = 0.f;
            for (int gidx = 0; gidx < kGroups; ++gidx) t += red[gidx * (G * K * 2 * V) + e];
            a.dw[static_cast<int64_t>(blockIdx.x) * a.d + o] = t;
        }
    }
}

// dweight[o] = sum over the CTAs' partial sums, in 64 bits: one warp a feature.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_dweight_kernel(const float* partial, int rows, int d, T* dweight)
{
    const int o = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (o >= d) return;
    double t = 0.0;
    for (int r = lane; r < rows; r += 32) t += static_cast<double>(partial[static_cast<int64_t>(r) * d + o]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) t += __shfl_xor_sync(kFull, t, k);
    if (lane == 0) dweight[o] = from_f<T>(static_cast<float>(t));
}

template <typename T, int V, int G, int K, bool GRAD>
void launch(const RotArgs& a, int grid, cudaStream_t s)
{
    norm_rotate_kernel<T, V, G, K, GRAD><<<grid, kThreads, 0, s>>>(a);
    count_launch();
}

template <typename T, int V, bool GRAD>
bool launch_v(const RotArgs& a, int G, int grid, cudaStream_t s)
{
    switch (G) {
        case 1: launch<T, V, 1, 1, GRAD>(a, grid, s); return true;
        case 2: launch<T, V, 2, 1, GRAD>(a, grid, s); return true;
        case 4: launch<T, V, 4, 1, GRAD>(a, grid, s); return true;
        case 8: launch<T, V, 8, 1, GRAD>(a, grid, s); return true;
        case 16: launch<T, V, 16, 1, GRAD>(a, grid, s); return true;
        case 32: launch<T, V, 32, 1, GRAD>(a, grid, s); return true;
    }
    return false;
}

// Turns per position of each pair, kept for the last (base, rotary) of the thread: 128 pow calls cost more
// than a launch.
void fill_turns(RotArgs& a, double base)
{
    static thread_local double last_base = 0.0;
    static thread_local int last_rotary = -1;
    static thread_local double table[kMaxPairs];
    if (last_base != base || last_rotary != a.rotary) {
        for (int p = 0; p < a.rotary / 2; ++p)
            table[p] = std::pow(base, -2.0 * p / a.rotary) / 6.283185307179586476925;
        last_base = base;
        last_rotary = a.rotary;
    }
    for (int p = 0; p < kMaxPairs; ++p) a.turns[p] = p < a.rotary / 2 ? table[p] : 0.0;
}

// The widest vectors that every row of x (and dy) allows: V features of 16 bytes, or 8.
template <typename T, bool GRAD>
sdtw_status run(RotArgs& a, void* dweight, cudaStream_t s)
{
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<sdtw_status>(e);
    const auto fits = [&](int V) {
        const int64_t bytes = V * static_cast<int64_t>(sizeof(T));
        uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                         static_cast<uintptr_t>((a.sb | a.sn | a.sh) * static_cast<int64_t>(sizeof(T)));
        if (GRAD)
            bits |= reinterpret_cast<uintptr_t>(a.dy) |
                    static_cast<uintptr_t>((a.gb | a.gn | a.gh) * static_cast<int64_t>(sizeof(T)));
        return a.d % (2 * V) == 0 && a.rotary % (2 * V) == 0 && bits % bytes == 0;
    };
    constexpr int kWide = 16 / sizeof(T);
    const int V = fits(kWide) ? kWide : (fits(4) ? 4 : 1);
    int G = 32;
    if (V > 1)
        for (G = 1; G * 2 * V < a.d;) G *= 2;
    // Heads a unit: all of a token's, so that they share its angles, unless that leaves lanes of the GPU idle.
    a.hpu = a.H;
    const int64_t groups = static_cast<int64_t>(sms) * kCtasPerSm * (kThreads / G);
    while (a.hpu > 1 && a.tokens * ((a.H + a.hpu - 1) / a.hpu) < 2 * groups) a.hpu = (a.hpu + 1) / 2;
    a.units_per_token = (a.H + a.hpu - 1) / a.hpu;
    const int64_t units = a.tokens * a.units_per_token;
    const int64_t need = (units + kThreads / G - 1) / (kThreads / G);
    int64_t grid = sms * static_cast<int64_t>(kCtasPerSm);
    if (grid > kMaxGradCtas) grid = kMaxGradCtas;
    if (grid > need) grid = need;
    if (V == 1)
        launch<T, 1, 32, 4, GRAD>(a, static_cast<int>(grid), s);
    else if (V == 4)
        launch_v<T, 4, GRAD>(a, G, static_cast<int>(grid), s);
    else
        launch_v<T, kWide, GRAD>(a, G, static_cast<int>(grid), s);
    if (GRAD && dweight != nullptr) {
        const int ctas = (a.d + kThreads / 32 - 1) / (kThreads / 32);
        if (a.weight_f32)
            join_dweight_kernel<float><<<ctas, kThreads, 0, s>>>(a.dw, static_cast<int>(grid), a.d,
                                                                 static_cast<float*>(dweight));
        else
            join_dweight_kernel<T><<<ctas, kThreads, 0, s>>>(a.dw, static_cast<int>(grid), a.d,
                                                             static_cast<T*>(dweight));
        count_launch();
    }
    e = cudaGetLastError();
    return e == cudaSuccess ? SDTW_OK : static_cast<sdtw_status>(e);
}

sdtw_status checked(const sdtw_rotate_problem* p, const void* y, bool grad, const void* dy, const void* dweight,
                    const void* ws, size_t ws_bytes)
{
    if (p == nullptr) return SDTW_EINVAL;
    if (p->dtype != SDTW_F32 && p->dtype != SDTW_F16 && p->dtype != SDTW_BF16) return SDTW_EDTYPE;
    if (p->B < 0 || p->N < 0 || p->H < 0 || p->d < 1 || p->d > 2 * kMaxPairs || p->H > (1 << 24)) return SDTW_EINVAL;
    if (p->rotary < 0 || p->rotary > p->d || p->rotary % 2 != 0 || !(p->base > 0) || !(p->eps >= 0)) return SDTW_EINVAL;
    if (p->position_kind < 0 || p->position_kind > 2) return SDTW_EINVAL;
    const bool empty = p->B == 0 || p->N == 0 || p->H == 0;
    if (!empty && (p->x == nullptr || y == nullptr || (grad && dy == nullptr) || p->err_word == nullptr)) return SDTW_EINVAL;
    if (dweight != nullptr && (ws == nullptr || ws_bytes < sdtw_norm_rotate_backward_workspace_bytes(p->d)))
        return SDTW_EWORKSPACE;
    return SDTW_OK;
}

void fill(RotArgs& a, const sdtw_rotate_problem* p)
{
    a.x = p->x;
    a.sb = p->x_stride[0];
    a.sn = p->x_stride[1];
    a.sh = p->x_stride[2];
    a.weight = p->weight;
    a.weight_f32 = p->weight_f32 || p->dtype == SDTW_F32;
    a.positions = p->positions;
    a.pos_kind = p->position_kind;
    a.pb = p->position_stride[0];
    a.pn = p->position_stride[1];
    a.len = {p->lengths, p->lengths_int32};
    a.err = p->err_word;
    a.tokens = p->B * p->N;
    a.N = p->N;
    a.H = static_cast<int>(p->H);
    a.d = static_cast<int>(p->d);
    a.rotary = static_cast<int>(p->rotary);
    a.interleaved = p->interleaved;
    a.eps = static_cast<float>(p->eps);
    fill_turns(a, p->base);
}

}  // namespace
}  // namespace sdtw

extern "C" {

size_t sdtw_norm_rotate_backward_workspace_bytes(int64_t d)
{
    return static_cast<size_t>(d) * sdtw::kMaxGradCtas * sizeof(float);
}

sdtw_status sdtw_norm_rotate(const sdtw_rotate_problem* p, void* y, void* stream)
{
    using namespace sdtw;
    const sdtw_status st = checked(p, y, false, nullptr, nullptr, nullptr, 0);
    if (st != SDTW_OK || p->B == 0 || p->N == 0 || p->H == 0) return st;
    RotArgs a{};
    fill(a, p);
    a.y = y;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p->dtype == SDTW_F32) return run<float, false>(a, nullptr, s);
    if (p->dtype == SDTW_F16) return run<__half, false>(a, nullptr, s);
    return run<__nv_bfloat16, false>(a, nullptr, s);
}

sdtw_status sdtw_norm_rotate_backward(const sdtw_rotate_problem* p, const void* dy, const int64_t* dy_stride, void* dx,
                                      void* dweight, void* workspace, size_t workspace_bytes, void* stream)
{
    using namespace sdtw;
    const sdtw_status st = checked(p, dx, true, dy, dweight, workspace, workspace_bytes);
    if (st != SDTW_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p->B == 0 || p->N == 0 || p->H == 0) {
        if (dweight == nullptr) return SDTW_OK;
        const size_t es = p->weight_f32 || p->dtype == SDTW_F32 ? 4 : 2;
        return static_cast<sdtw_status>(cudaMemsetAsync(dweight, 0, es * static_cast<size_t>(p->d), s));
    }
    if (dy_stride == nullptr) return SDTW_EINVAL;
    RotArgs a{};
    fill(a, p);
    a.dy = dy;
    a.gb = dy_stride[0];
    a.gn = dy_stride[1];
    a.gh = dy_stride[2];
    a.y = dx;
    a.dw = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
    if (p->dtype == SDTW_F32) return run<float, true>(a, dweight, s);
    if (p->dtype == SDTW_F16) return run<__half, true>(a, dweight, s);
    return run<__nv_bfloat16, true>(a, dweight, s);
}

}  // extern "C"
