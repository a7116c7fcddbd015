// Gradients of cross attention on warp-level mma: float32, and 16-bit operands of any alignment. Two launches, dq by tiles of
// queries and then dk and dv by tiles of states, with the formulas of the tensor-core kernels (sdtw_attention_tc_bwd.cu) and
// like them without atomics on results. One kernel serves both: the tile's rows (Q, dO; or K, V) stay in shared memory, 16 a
// warp, and the other side streams past in tiles of TC rows:
//   S = X1 Y1^T, dP = X2 Y2^T;   dq: sum dS Y1;   dk: sum dS Y1, dv: sum P Y2.
// float32 is bound by the instructions that split operands into heads and tails, once for each use: 64 x 256 x 192 x 4 x 32,
// band 32, 135 us; 2 x 2048 x 2048 x 8 x 128 3.55 ms, 34 TFLOP/s of the seven products. 16-bit operands of odd width, by their copies of
// two bytes: 32 x 512 x 512 x 8 x 33 bf16 1.03 ms, against 0.12 for 40 features on tcgen05.
#include "sdtw_attention_mma.cuh"
#include "sdtw_attention_range.cuh"
#include "sdtw_attention_split.h"

namespace sdtw {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16 * kWarps;

template <typename T>
constexpr bool is_half = std::is_same<T, __half>::value;

template <typename T, int DPAD>
struct Geom {
    static constexpr int TC = sizeof(T) == 4 && DPAD == 128 ? 16 : 32;
    // CTAs an SM, registers given up for them: fp32, d = 32: 144 -> 136 us; d = 128: 3.69 -> 3.54 ms
    static constexpr int CTAS = sizeof(T) == 4 && DPAD == 32 ? 4 : 2;
    static constexpr int UNIT = 16 / sizeof(T);
    static constexpr int LD = DPAD + UNIT;
    static constexpr int STAGES = 2;
    static constexpr int OFF_X2 = kRows * LD;  // elements
    static constexpr int OFF_RING = 2 * kRows * LD;
    static constexpr int TILE = TC * LD;
    static constexpr int OFF_STAT = (OFF_RING + STAGES * 2 * TILE) * static_cast<int>(sizeof(T));  // bytes
    static constexpr int BYTES = OFF_STAT + 4 * (STAGES * 2 * TC + 2 * kRows);
};

struct Args {
    AttnArgs a;
    int tiles;  // CTAs a head
};

template <typename T, int DPAD, int VB, bool KV>
__global__ void __launch_bounds__(kThreads, Geom<T, DPAD>::CTAS) attend_backward_mma_kernel(const __grid_constant__ Args f)
{
    using G = Geom<T, DPAD>;
    constexpr int UPR = DPAD / G::UNIT;
    constexpr float kShift = is_half<T> ? kHalfShift : 0.f, kUnshift = is_half<T> ? kHalfUnshift : 1.f;
    const AttnArgs& a = f.a;
    extern __shared__ __align__(128) unsigned char sm[];
    T* x1 = reinterpret_cast<T*>(sm);
    T* x2 = x1 + G::OFF_X2;
    T* ring = x1 + G::OFF_RING;
    float* col_stat = reinterpret_cast<float*>(sm + G::OFF_STAT);  // KV: STAGES of (lse, delta) of TC queries
    float* row_stat = col_stat + G::STAGES * 2 * G::TC;            // dq: delta and |do|^2 of the rows
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int H = KV ? a.Hkv : a.Hq;
    const int tile = static_cast<int>(blockIdx.x % f.tiles);
    const int hr = static_cast<int>(blockIdx.x / f.tiles % H), b = static_cast<int>(blockIdx.x / f.tiles / H);
    const int hk = KV ? hr : hr / a.group;
    const int64_t row0 = static_cast<int64_t>(tile) * kRows;
    int64_t nx, ny;
    if (!pair_lengths(a, b, nx, ny) && tid == 0) atomicOr(a.err, kErrBadLength);
    const int64_t nr = KV ? ny : nx, nc = KV ? nx : ny;  // lengths of the rows' and the columns' series
    const int64_t all_rows = KV ? a.M : a.N;
    const auto cells = [&](int64_t r, int64_t& lo, int64_t& hi) {
        if (KV)
            column_cells(a, r, nx, ny, lo, hi);
        else
            row_cells(a, r, nx, ny, lo, hi);
    };
    int64_t c0 = 0, c1 = 0;
    if (row0 < nr && nc > 0) {
        int64_t dummy;
        cells(row0, c0, dummy);
        cells((row0 + kRows < nr ? row0 + kRows : nr) - 1, dummy, c1);
    }
    const int per_head = static_cast<int>((c1 - c0 + G::TC - 1) / G::TC);
    const int steps = KV ? per_head * a.group : per_head;
    int64_t lo[2] = {0, 0}, hi[2] = {0, 0};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int64_t r = row0 + warp * 16 + (lane >> 2) + 8 * x;
        if (r < nr && nc > 0) cells(r, lo[x], hi[x]);
    }

    const Strides &r1s = KV ? a.ks : a.qs, &r2s = KV ? a.vs : a.gs, &y1s = KV ? a.qs : a.ks, &y2s = KV ? a.gs : a.vs;
    const T* r1p = static_cast<const T*>(KV ? a.k : a.q) + b * r1s.b + hr * r1s.h;
    const T* r2p = static_cast<const T*>(KV ? a.v : a.dout) + b * r2s.b + hr * r2s.h;
    float gscale = 1.f;  // of dS: here for all states of the CTA, in dq a row's own
    if (is_half<T> && KV && c1 > c0)
        gscale = half_scale(gradient_bound(a, b, hk, c0, c1, row0, row0 + kRows < nr ? row0 + kRows : nr));
    const float cf = gscale * kUnshift;

    const auto load_tile = [&](int t) {
        const int h = KV ? hk * a.group + t / per_head : hk;
        const int64_t c = c0 + static_cast<int64_t>(KV ? t % per_head : t) * G::TC;
        const T* y1p = static_cast<const T*>(KV ? a.q : a.k) + b * y1s.b + h * y1s.h;
        const T* y2p = static_cast<const T*>(KV ? a.dout : a.v) + b * y2s.b + h * y2s.h;
        T* to = ring + t % G::STAGES * 2 * G::TILE;
        const int u = tid % UPR;
        if (u * G::UNIT < a.d)
#pragma unroll
            for (int r = tid / UPR; r < G::TC; r += kThreads / UPR) {
                const bool on = c + r < nc;
                const int64_t row = on ? c + r : c0;
                copy_unit<T, VB>(to + r * G::LD + u * G::UNIT, y1p + row * y1s.n + u * G::UNIT, u * G::UNIT, a.d, on);
                copy_unit<T, VB>(to + G::TILE + r * G::LD + u * G::UNIT, y2p + row * y2s.n + u * G::UNIT, u * G::UNIT, a.d, on);
            }
        if (KV && tid < G::TC) {
            const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.N + c + tid;
            const bool on = c + tid < nc;
            float* st = col_stat + t % G::STAGES * 2 * G::TC;
            st[tid] = on ? kShift - a.lse[at] : -INFINITY;  // P = 2^-inf past the length
            st[G::TC + tid] = on ? a.delta[at] * cf : 0.f;
        }
    };
    if (a.d < DPAD) {  // features from d to DPAD are zero in every buffer
        const int tail = DPAD - a.d;
        for (int e = tid; e < (2 * kRows + G::STAGES * 2 * G::TC) * tail; e += kThreads)
            x1[e / tail * G::LD + a.d + e % tail] = from_f<T>(0.f);
    }
    {
        const int u = tid % UPR;
        if (u * G::UNIT < a.d)
            for (int r = tid / UPR; r < kRows; r += kThreads / UPR) {
                const bool on = row0 + r < nr;
                const int64_t row = on ? row0 + r : 0;
                copy_unit<T, VB>(x1 + r * G::LD + u * G::UNIT, r1p + row * r1s.n + u * G::UNIT, u * G::UNIT, a.d, on);
                copy_unit<T, VB>(x2 + r * G::LD + u * G::UNIT, r2p + row * r2s.n + u * G::UNIT, u * G::UNIT, a.d, on);
            }
    }
    if (steps > 0) load_tile(0);
    cp_async_commit();
    PeakPart v_part{};  // of the largest |v| of the CTA's states
    if (is_half<T> && !KV && c1 > c0) v_part = value_part(a, b, hk, c0, c1);
    if constexpr (!KV) {
        // delta and |do|^2 of this warp's rows.
        float top_delta = 0.f, top_norm = 0.f;
        for (int r = warp * 16; r < warp * 16 + 16; ++r) {
            const int64_t i = row0 + r;
            float dot = 0.f, nrm = 0.f;
            if (i < nx && ny > 0) {
                const int64_t at = ((static_cast<int64_t>(b) * a.N + i) * a.Hq + hr) * a.d;
                for (int c = lane; c < a.d; c += 32) {
                    const float g = to_f(r2p[i * r2s.n + c]);
                    float o = to_f(static_cast<const T*>(a.o)[at + c]);
                    if (a.o_lo) o = fmaf(to_f(static_cast<const T*>(a.o_lo)[at + c]), 1.f / kLoScale<T>, o);
                    dot = fmaf(g, o, dot);
                    nrm = fmaf(g, g, nrm);
                }
            }
            dot = warp_sum(dot);
            nrm = warp_sum(nrm);
            if (lane == 0) {
                row_stat[r] = dot;
                row_stat[kRows + r] = nrm;
                if (i < a.N) a.delta[(static_cast<int64_t>(b) * a.Hq + hr) * a.N + i] = dot;
            }
            top_delta = fmaxf(top_delta, fabsf(dot));
            top_norm = fmaxf(top_norm, nrm);
        }
        if (is_half<T> && lane == 0 && row0 + warp * 16 < nx) raise_gradient_peak(a, b, hk, row0 + warp * 16, top_norm, top_delta);
        __syncwarp();
    }
    float r_bias[2], r_delta[2], r_scale[2], r_cf[2];  // dq: of this thread's rows
    float v_top = 0.f;
    if constexpr (is_half<T> && !KV) v_top = peak_of(v_part);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = warp * 16 + (lane >> 2) + 8 * x;
        r_scale[x] = is_half<T> && !KV ? half_scale(fmaf(sqrtf(row_stat[kRows + r]), v_top, fabsf(row_stat[r]))) : gscale;
        r_cf[x] = is_half<T> && !KV ? r_scale[x] * kUnshift : cf;
        r_delta[x] = KV ? 0.f : row_stat[r] * r_cf[x];
        r_bias[x] = !KV && hi[x] > lo[x] ? kShift - a.lse[(static_cast<int64_t>(b) * a.Hq + hr) * a.N + row0 + r] : -INFINITY;
    }

    float acc1[DPAD / 8][4], acc2[KV ? DPAD / 8 : 1][4];
#pragma unroll
    for (int x = 0; x < DPAD / 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc1[x][e] = 0.f;
            if constexpr (KV) acc2[x][e] = 0.f;
        }
    for (int t = 0; t < steps; ++t) {
        cp_async_wait<0>();
        __syncthreads();
        if (t + 1 < steps) load_tile(t + 1);
        cp_async_commit();
        const T* y1 = ring + t % G::STAGES * 2 * G::TILE;
        const T* y2 = y1 + G::TILE;
        const float* st = col_stat + t % G::STAGES * 2 * G::TC;
        const int64_t c = c0 + static_cast<int64_t>(KV ? t % per_head : t) * G::TC;
        // A warp passes over tiles without a cell of its rows (those of a band are not those of its CTA).
        const bool some = (c < hi[0] && c + G::TC > lo[0]) || (c < hi[1] && c + G::TC > lo[1]);
        if (!__any_sync(kFull, some)) continue;
        float s[G::TC / 8][4], dp[G::TC / 8][4];
#pragma unroll
        for (int x = 0; x < G::TC / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][e] = dp[x][e] = 0.f;
        product_rows<T, DPAD, G::LD, G::TC / 8>(s, x1 + warp * 16 * G::LD, y1, lane);
        product_rows<T, DPAD, G::LD, G::TC / 8>(dp, x2 + warp * 16 * G::LD, y2, lane);
        const bool whole = __all_sync(kFull, c >= lo[0] && c >= lo[1] && c + G::TC <= hi[0] && c + G::TC <= hi[1]);
#pragma unroll
        for (int x = 0; x < G::TC / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 8 * x + 2 * (lane & 3) + (e & 1), row = e >> 1;
                const float bias = KV ? st[col] : r_bias[row], delta = KV ? st[G::TC + col] : r_delta[row];
                float p = ex2f(fmaf(s[x][e], a.scale_log2, bias));
                if (!whole && (c + col < lo[row] || c + col >= hi[row])) p = 0.f;
                s[x][e] = p;
                dp[x][e] = p * fmaf(dp[x][e], is_half<T> ? r_cf[row] : 1.f, -delta);
            }
        product_columns<T, DPAD, G::LD, G::TC / 8>(acc1, dp, y1, lane);
        // dq of few features: what the rounding of dS dropped goes through a second product (as in the tensor-core kernel).
        if constexpr (!KV && sizeof(T) == 2 && DPAD == 32) {
#pragma unroll
            for (int x = 0; x < G::TC / 8; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[x][e] -= to_f(from_f<T>(dp[x][e]));
            product_columns<T, DPAD, G::LD, G::TC / 8>(acc1, dp, y1, lane);
        }
        if constexpr (KV) product_columns<T, DPAD, G::LD, G::TC / 8>(acc2, s, y2, lane);
    }
    cp_async_wait<0>();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int64_t r = row0 + warp * 16 + (lane >> 2) + 8 * x;
        if (r >= all_rows) continue;
        const int64_t at = ((static_cast<int64_t>(b) * all_rows + r) * H + hr) * a.d;
        const float back = a.scale / r_scale[x];
        const bool any = hi[x] > lo[x];
        T* out1 = static_cast<T*>(KV ? a.dk : a.dq) + at;
        T* out2 = static_cast<T*>(a.dv) + at;
#pragma unroll
        for (int y = 0; y < DPAD / 8; ++y)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * y + 2 * (lane & 3) + e;
                if (col >= a.d) continue;
                out1[col] = from_f<T>(any ? acc1[y][2 * x + e] * back : 0.f);
                if constexpr (KV) out2[col] = from_f<T>(any ? acc2[y][2 * x + e] * kUnshift : 0.f);
            }
    }
}

template <typename T, int DPAD, int VB>
cudaError_t launch(Args& f, cudaStream_t s)
{
    using G = Geom<T, DPAD>;
    static_assert(G::CTAS * (G::BYTES + 1024) <= 228 * 1024, "the CTAs of an SM");
    const auto dq = attend_backward_mma_kernel<T, DPAD, VB, false>;
    const auto dkv = attend_backward_mma_kernel<T, DPAD, VB, true>;
    static std::atomic<bool> allowed[2][128];
    cudaError_t e = allow_smem(dq, G::BYTES, allowed[0]);
    if (e == cudaSuccess) e = allow_smem(dkv, G::BYTES, allowed[1]);
    if (e != cudaSuccess) return e;
    if (f.a.N > 0) {
        f.tiles = static_cast<int>((f.a.N + kRows - 1) / kRows);
        dq<<<static_cast<unsigned>(static_cast<int64_t>(f.a.B) * f.a.Hq * f.tiles), kThreads, G::BYTES, s>>>(f);
        count_launch();
    }
    if (f.a.M > 0) {
        f.tiles = static_cast<int>((f.a.M + kRows - 1) / kRows);
        dkv<<<static_cast<unsigned>(static_cast<int64_t>(f.a.B) * f.a.Hkv * f.tiles), kThreads, G::BYTES, s>>>(f);
        count_launch();
    }
    return cudaGetLastError();
}

template <typename T, int DPAD>
cudaError_t launch_vb(Args& f, int vb, cudaStream_t s)
{
    if (vb == 16) return launch<T, DPAD, 16>(f, s);
    if (vb >= 4) return launch<T, DPAD, 4>(f, s);
    if constexpr (sizeof(T) == 2) return launch<T, DPAD, 2>(f, s);
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t backward_t(Args& f, cudaStream_t s)
{
    const AttnArgs& a = f.a;
    const int vb = copy_bytes(step_bits<T>(a.q, a.qs) | step_bits<T>(a.k, a.ks) | step_bits<T>(a.v, a.vs) |
                              step_bits<T>(a.dout, a.gs) | a.d * sizeof(T));
    if (a.d <= 32) return launch_vb<T, 32>(f, vb, s);
    if (a.d <= 64) return launch_vb<T, 64>(f, vb, s);
    return launch_vb<T, 128>(f, vb, s);
}

}  // namespace

cudaError_t attention_mma_backward(const AttnArgs& a, int dtype, cudaStream_t s)
{
    Args f{};
    f.a = a;
    if (dtype == SDTW_F16) return backward_t<__half>(f, s);
    return dtype == SDTW_F32 ? backward_t<float>(f, s) : backward_t<__nv_bfloat16>(f, s);
}

}  // namespace sdtw
