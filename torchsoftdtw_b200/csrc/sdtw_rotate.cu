// RMS norm of every head followed by the rotation of its features by the position, and the gradient:
//   r = (mean(x^2) + eps)^(-1/2),  u = x r,  z = u w,  y = R z
//   R turns the pair p = 0 .. rotary/2 - 1 of z by the angle pos * base^(-2p / rotary); pairs are the features
//   (p, p + rotary/2), or (2p, 2p + 1) when interleaved; the features from `rotary` on stay.
//   backward: g = R^T dy, dw = sum g u, dx = r (g w - u mean(g w u)); r is formed again from x.
//
// Bound by memory: x in and y out; x and dy in, dx out. A head (d features) belongs to a group of G lanes, a
// lane to V neighbouring pairs (two vectors of V features), so the mean is log2 G shuffles and a pair never
// leaves its lane. A unit of work is `hpu` heads of one token, whose angles are formed once (64-bit products, so that far
// positions keep theirs); units go round the groups, so that the GPU sweeps memory in order, and a group loads U heads ahead
// of their arithmetic. dw: every lane adds the products of its own features over its run in 32 bits,
// the CTA joins its groups, a second launch joins the CTAs, each in a fixed order.
#include <cmath>
#include <mutex>

#include "sdtw_sequence.cuh"

namespace sdtw {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // d <= 256
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
    int hpu, token_units;  // heads a unit, units a token
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

// Features of pair group `pg` (V pairs from p0 = pg V): where its two vectors of V features begin, and whether it turns.
// The host only chooses V > 1 when V divides rotary / 2 and 2 V divides d, so a group is all of one kind. Pairs that turn are
// the two vectors' features side by side in the split layout (`apart`); in the interleaved one, and for features that
// stay, the two vectors are 2V neighbours and a pair is two of those.
template <int V, bool SPLIT>
__device__ __forceinline__ void pair_offsets(const RotArgs& a, int pg, int& oa, int& ob, bool& turned)
{
    const int p0 = pg * V, half = a.rotary / 2;
    turned = p0 < half;
    if (SPLIT && turned) {
        oa = p0;
        ob = p0 + half;
    } else {
        oa = 2 * p0;
        ob = 2 * p0 + V;
    }
}
// Place of the first (second) feature of pair i of a group among its 2V features, the second vector from V on.
template <int V, bool SPLIT>
__device__ __forceinline__ constexpr int place(int i, bool second)
{
    return SPLIT ? (second ? V + i : i) : 2 * i + (second ? 1 : 0);
}

// Two numbers in one instruction.
struct F2 {
    float x, y;
};
__device__ __forceinline__ uint64_t bits(F2 a)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ F2 both(uint64_t r)
{
    F2 a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
    return a;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return both(r);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return both(r);
}
__device__ __forceinline__ F2 twice(float a) { return {a, a}; }
__device__ __forceinline__ F2 minus(F2 a) { return {-a.x, -a.y}; }

// The features of one head that a lane holds, as they lie in memory: K groups of two vectors.
template <typename T, int V, int K>
struct Raw {
    Vec<T, V> v[K][2];
};

template <typename T, int V, int K>
__device__ __forceinline__ void load_raw(Raw<T, V, K>& r, const T* row, const int (&oa)[K], const int (&ob)[K], const bool (&live)[K],
                                         int d, bool on)
{
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[k][0].e[i] = r.v[k][1].e[i] = from_f<T>(0.f);
        if (on && live[k]) {
            if constexpr (V == 1) {
                if (oa[k] < d) r.v[k][0].e[0] = row[oa[k]];
                if (ob[k] < d) r.v[k][1].e[0] = row[ob[k]];
            } else {
                r.v[k][0] = *reinterpret_cast<const Vec<T, V>*>(row + oa[k]);
                r.v[k][1] = *reinterpret_cast<const Vec<T, V>*>(row + ob[k]);
            }
        }
    }
}
template <typename T, int V, int K>
__device__ __forceinline__ void store_raw(const Raw<T, V, K>& r, T* row, const int (&oa)[K], const int (&ob)[K], const bool (&live)[K],
                                          int d, bool on)
{
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!on || !live[k]) continue;
        if constexpr (V == 1) {
            if (oa[k] < d) row[oa[k]] = r.v[k][0].e[0];
            if (ob[k] < d) row[ob[k]] = r.v[k][1].e[0];
        } else {
            *reinterpret_cast<Vec<T, V>*>(row + oa[k]) = r.v[k][0];
            *reinterpret_cast<Vec<T, V>*>(row + ob[k]) = r.v[k][1];
        }
    }
}

// Two neighbouring 16-bit features as floats, and back in one conversion.
__device__ __forceinline__ F2 two_f(const __half* e)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(e));
    return {f.x, f.y};
}
__device__ __forceinline__ F2 two_f(const __nv_bfloat16* e)
{
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(e));
    return {f.x, f.y};
}
__device__ __forceinline__ void put_two(__half* e, F2 f) { *reinterpret_cast<__half2*>(e) = __floats2half2_rn(f.x, f.y); }
__device__ __forceinline__ void put_two(__nv_bfloat16* e, F2 f)
{
    *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(f.x, f.y);
}

// A lane's pairs, two by two: the firsts in p, the seconds in q (V K pairs, an even number).
template <typename T, int V, int K, bool SPLIT>
__device__ __forceinline__ void unpack(const Raw<T, V, K>& r, F2 (&p)[V * K / 2], F2 (&q)[V * K / 2])
{
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if constexpr (SPLIT) {
                p[i] = two_f(r.v[0][0].e + 2 * i);
                q[i] = two_f(r.v[0][1].e + 2 * i);
            } else {  // features 4i .. 4i + 3: first, second, first, second
                const F2 a = two_f(r.v[0][4 * i / V].e + 4 * i % V), b = two_f(r.v[0][(4 * i + 2) / V].e + (4 * i + 2) % V);
                p[i] = {a.x, b.x};
                q[i] = {a.y, b.y};
            }
        }
    } else {
        const auto at = [&](int pair, bool second) {
            const int k = pair / V, o = place<V, SPLIT>(pair % V, second);
            return to_f(o < V ? r.v[k][0].e[o] : r.v[k][1].e[o - V]);
        };
#pragma unroll
        for (int i = 0; i < V * K / 2; ++i) {
            p[i] = {at(2 * i, false), at(2 * i + 1, false)};
            q[i] = {at(2 * i, true), at(2 * i + 1, true)};
        }
    }
}
template <typename T, int V, int K, bool SPLIT>
__device__ __forceinline__ void repack(Raw<T, V, K>& r, const F2 (&p)[V * K / 2], const F2 (&q)[V * K / 2])
{
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if constexpr (SPLIT) {
                put_two(r.v[0][0].e + 2 * i, p[i]);
                put_two(r.v[0][1].e + 2 * i, q[i]);
            } else {
                put_two(r.v[0][4 * i / V].e + 4 * i % V, {p[i].x, q[i].x});
                put_two(r.v[0][(4 * i + 2) / V].e + (4 * i + 2) % V, {p[i].y, q[i].y});
            }
        }
    } else {
        const auto put = [&](int pair, bool second, float x) {
            const int k = pair / V, o = place<V, SPLIT>(pair % V, second);
            (o < V ? r.v[k][0].e[o] : r.v[k][1].e[o - V]) = from_f<T>(x);
        };
#pragma unroll
        for (int i = 0; i < V * K / 2; ++i) {
            put(2 * i, false, p[i].x);
            put(2 * i + 1, false, p[i].y);
            put(2 * i, true, q[i].x);
            put(2 * i + 1, true, q[i].y);
        }
    }
}

// How many heads a lane has in flight, and how many CTAs of an SM the registers that this takes leave room for. Measured,
// 16 x 4096 x 16 x 128 bf16 (V = 8): forward 97 us with four heads and two CTAs, 126 with two and three; gradient 179 with
// one, 204 with two. 32 x 512 x 8 x 64 float32 (V = 4): forward 17.4 with two and three, 19.5 with four and two.
template <int V, bool GRAD>
constexpr int kAhead = V == 1 ? 1 : (V == 8 ? (GRAD ? 1 : 4) : 2);
template <int V, bool GRAD>
constexpr int kCtasPerSm = V == 8 || GRAD ? 2 : 3;

// cos and sin of `turns` whole turns, |turns| <= 1/2. 16-bit results: the hardware's functions, off by at most 2^-21 on
// [-pi, pi], far below half a step of y and dx. A float32 dweight of 16-bit x takes them too: its sums over tokens are held in
// 32 bits a lane and carry as much (the full functions in the gradient: 128 us instead of 121, 8 x 4097 x 13 x 96 fp16).
template <typename T>
__device__ __forceinline__ void cos_sin(float turns, float& c, float& s)
{
    if constexpr (sizeof(T) == 2)
        __sincosf(turns * 6.283185307179586f, &s, &c);
    else
        sincospif(2.f * turns, &s, &c);
}

// K pair groups a lane (1, or 4 with V = 1 and G = 32: any d up to 256, odd or unaligned).
template <typename T, int V, int G, int K, bool SPLIT, bool GRAD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm<V, GRAD>) norm_rotate_kernel(const __grid_constant__ RotArgs a)
{
    constexpr int kGroups = kThreads / G;
    constexpr int U = kAhead<V, GRAD>;
    constexpr int NP = V * K / 2;  // twos of pairs
    __shared__ float red[GRAD ? kGroups * G * K * 2 * V : 1];
    const int gl = threadIdx.x % G, group = threadIdx.x / G;
    const int pair_groups = (a.d + 2 * V - 1) / (2 * V);
    int oa[K], ob[K];
    bool turned[K], live[K];
    F2 wp[NP], wq[NP], dwp[NP], dwq[NP];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        live[k] = gl + k * G < pair_groups;
        pair_offsets<V, SPLIT>(a, live[k] ? gl + k * G : 0, oa[k], ob[k], turned[k]);
        turned[k] = turned[k] && live[k];
    }
    // Vector o of group k holds feature (o < V ? oa : ob - V) + o.
    const auto feature = [&](int pair, bool second) {
        const int o = place<V, SPLIT>(pair % V, second);
        return (o < V ? oa[pair / V] : ob[pair / V] - V) + o;
    };
    const auto weight_at = [&](int pair, bool second) {
        const int o = feature(pair, second);
        if (a.weight == nullptr || !live[pair / V] || o >= a.d) return 1.f;
        return a.weight_f32 ? static_cast<const float*>(a.weight)[o] : to_f(static_cast<const T*>(a.weight)[o]);
    };
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        wp[i] = {weight_at(2 * i, false), weight_at(2 * i + 1, false)};
        wq[i] = {weight_at(2 * i, true), weight_at(2 * i + 1, true)};
        dwp[i] = dwq[i] = {0.f, 0.f};
    }
    const float inv_d = 1.f / static_cast<float>(a.d);
    const int64_t units = a.tokens * a.token_units, stride = static_cast<int64_t>(gridDim.x) * kGroups;
    // Every lane of a warp makes the same number of rounds (the shuffles need them all).
    for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * kGroups; u0 < units; u0 += stride) {
        const bool on = u0 + group < units;
        const unsigned unit = static_cast<unsigned>(on ? u0 + group : 0);  // fewer than 2^31, as the host checks
        const unsigned token = unit / static_cast<unsigned>(a.token_units), b = token / static_cast<unsigned>(a.N);
        const int64_t n = token - b * static_cast<unsigned>(a.N);
        const int first = static_cast<int>(unit - token * static_cast<unsigned>(a.token_units)) * a.hpu;
        const int last = on ? min(first + a.hpu, a.H) : first;
        const int64_t len = a.len.get(b, a.N);
        if (on && len < 0 && gl == 0) atomicOr(a.err, kErrBadLength);
        const bool work = on && n < len;
        const T* xr = static_cast<const T*>(a.x) + static_cast<int64_t>(b) * a.sb + n * a.sn + first * a.sh;
        const T* gr = GRAD ? static_cast<const T*>(a.dy) + static_cast<int64_t>(b) * a.gb + n * a.gn + first * a.gh : nullptr;
        T* yr = static_cast<T*>(a.y) + (static_cast<int64_t>(token) * a.H + first) * a.d;
        F2 c[NP], s[NP];
        bool fresh = true;
        for (int h0 = first; h0 < first + a.hpu; h0 += U) {
            Raw<T, V, K> rx[U], rg[GRAD ? U : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                load_raw<T, V, K>(rx[u], xr, oa, ob, live, a.d, work && h0 + u < last);
                xr += a.sh;
                if constexpr (GRAD) {
                    load_raw<T, V, K>(rg[u], gr, oa, ob, live, a.d, work && h0 + u < last);
                    gr += a.gh;
                }
            }
            if (fresh) {  // the angles, once a unit, behind its first loads
                const double pos = work ? position(a, b, n) : 0.0;
#pragma unroll
                for (int i = 0; i < 2 * NP; ++i) {
                    float ci = 1.f, si = 0.f;
                    if (turned[i / V]) {
                        const double t = pos * a.turns[(gl + i / V * G) * V + i % V];
                        cos_sin<T>(static_cast<float>(t - rint(t)), ci, si);  // turns beyond whole ones, in [-1/2, 1/2]
                    }
                    (i & 1 ? c[i / 2].y : c[i / 2].x) = ci;
                    (i & 1 ? s[i / 2].y : s[i / 2].x) = si;
                }
                fresh = false;
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                F2 p[NP], q[NP], ss2 = {0.f, 0.f};
                unpack<T, V, K, SPLIT>(rx[u], p, q);
#pragma unroll
                for (int i = 0; i < NP; ++i) ss2 = fma2(q[i], q[i], fma2(p[i], p[i], ss2));
                const float ss = group_sum<G>(ss2.x + ss2.y);
                // Rows that are not worked on were read as zeros and stay so; those of a bad sample become NaN.
                const float r = work ? rsqrtf(fmaf(ss, inv_d, a.eps)) : (len < 0 && !GRAD ? __int_as_float(0x7fc00000) : 0.f);
                Raw<T, V, K> ry;
                if constexpr (GRAD) {
                    F2 g[NP], e[NP], dot2 = {0.f, 0.f};
                    unpack<T, V, K, SPLIT>(rg[u], g, e);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {  // turned back
                        const F2 y0 = g[i], y1 = e[i];
                        g[i] = fma2(y1, s[i], y0 * c[i]);
                        e[i] = fma2(minus(y0), s[i], y1 * c[i]);
                    }
                    F2 gp[NP], gq[NP];
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        gp[i] = g[i] * p[i];
                        gq[i] = e[i] * q[i];
                        dot2 = fma2(gq[i], wq[i], fma2(gp[i], wp[i], dot2));
                    }
                    const float dot = group_sum<G>(dot2.x + dot2.y);
                    const F2 back = twice(-dot * inv_d * r * r * r), r2 = twice(r);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        dwp[i] = fma2(gp[i], r2, dwp[i]);
                        dwq[i] = fma2(gq[i], r2, dwq[i]);
                        p[i] = fma2(g[i] * wp[i], r2, p[i] * back);
                        q[i] = fma2(e[i] * wq[i], r2, q[i] * back);
                    }
                } else {
                    const F2 r2 = twice(r);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const F2 z0 = p[i] * r2 * wp[i], z1 = q[i] * r2 * wq[i];
                        p[i] = fma2(minus(z1), s[i], z0 * c[i]);
                        q[i] = fma2(z0, s[i], z1 * c[i]);
                    }
                }
                repack<T, V, K, SPLIT>(ry, p, q);
                store_raw<T, V, K>(ry, yr, oa, ob, live, a.d, h0 + u < last);
                yr += a.d;
            }
        }
    }
    if constexpr (GRAD) {
        if (a.dw == nullptr) return;
        // red[group][lane][pair][first, second]; then the features' sums over the groups, in order.
        float* mine = red + (group * G + gl) * (K * 2 * V);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            mine[4 * i] = dwp[i].x;
            mine[4 * i + 1] = dwq[i].x;
            mine[4 * i + 2] = dwp[i].y;
            mine[4 * i + 3] = dwq[i].y;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < G * K * 2 * V; e += kThreads) {
            const int lane = e / (K * 2 * V), pair = e / 2 % (K * V), pg = lane + pair / V * G;
            if (pg >= pair_groups) continue;
            int fa, fb;
            bool tn;
            pair_offsets<V, SPLIT>(a, pg, fa, fb, tn);
            const int at = place<V, SPLIT>(pair % V, e & 1);
            const int o = at < V ? fa + at : fb + at - V;
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
    if (a.interleaved)
        norm_rotate_kernel<T, V, G, K, false, GRAD><<<grid, kThreads, 0, s>>>(a);
    else
        norm_rotate_kernel<T, V, G, K, true, GRAD><<<grid, kThreads, 0, s>>>(a);
    count_launch();
}

template <typename T, int V, bool GRAD>
void launch_v(const RotArgs& a, int G, int grid, cudaStream_t s)
{
    switch (G) {
        case 1: launch<T, V, 1, 1, GRAD>(a, grid, s); break;
        case 2: launch<T, V, 2, 1, GRAD>(a, grid, s); break;
        case 4: launch<T, V, 4, 1, GRAD>(a, grid, s); break;
        case 8: launch<T, V, 8, 1, GRAD>(a, grid, s); break;
        case 16: launch<T, V, 16, 1, GRAD>(a, grid, s); break;
        default: launch<T, V, 32, 1, GRAD>(a, grid, s); break;
    }
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
    cudaError_t e = current_sms(dev, sms);
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
    // A unit is a token, unless that leaves the groups with few and unequal shares of them: then parts of one.
    const int64_t groups = static_cast<int64_t>(sms) * kCtasPerSm<kWide, GRAD> * (kThreads / G);
    a.hpu = a.H;
    while (a.hpu > 4 && a.tokens * ((a.H + a.hpu - 1) / a.hpu) < 8 * groups) a.hpu = (a.hpu + 7) / 8 * 4;
    if (a.tokens * a.H < groups) a.hpu = 1;
    a.token_units = (a.H + a.hpu - 1) / a.hpu;
    const int64_t units = a.tokens * a.token_units;
    if (units >= (int64_t{1} << 31)) return SDTW_EINVAL;
    int64_t grid = (units + kThreads / G - 1) / (kThreads / G);
    if (grid > sms * kCtasPerSm<kWide, GRAD>) grid = sms * kCtasPerSm<kWide, GRAD>;
    if (grid > kMaxGradCtas) grid = kMaxGradCtas;
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
