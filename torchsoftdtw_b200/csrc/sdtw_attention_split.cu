// Cross attention with the states of one sample split over CTAs: few query rows (decoded tokens), and float32.
//
// The N group query rows that read one key head are packed (row r is query r / group of head r % group): a CTA takes
// ROWS of them and one split of the states that their cells touch. K and V stream through a ring of cp.async tiles;
// products are warp-level mma (16-bit operands m16n8k16; float32 as three TF32 products of heads and tails). With
// ROWS = 16 the four warps take different states of each tile and join at the end; with ROWS = 64 each takes its own 16 rows
// and all states.
//
// Few rows are bound by reading K and V once, so the rows of a padded mma cost nothing; the splits exist to have every SM
// read. Up to eight splits form a cluster and join their sums through distributed shared memory, in one launch; more
// (a single sequence of few heads) leave partial sums in the workspace for a second launch. Both join in split order.
//
// Memory bound with few rows: 16 x 1 x 32771 x 32/8 x 128 bf16 379 us, 5.65 TB/s of 6.55 measured for a copy (two splits a head;
// three to eight 393 to 500 us). Short caches are bound by launch and latency: 8 x 1 x 512 x 8 x 64 10 us a call. A token's float32
// cache is read at 2.86 TB/s (1.51 ms for the same sizes): its operands are split for a product of 16 rows. float32 with
// many rows is bound by the instructions that split operands: 64 x 256 x 192 x 4 x 32, band 32, 49 us; 2 x 2048 x 2048 x 8 x 128
// 0.98 ms, 35 TFLOP/s (3 x 35 on the matrix pipe).
#include "sdtw_attention_mma.cuh"
#include "sdtw_attention_split.h"

namespace sdtw {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kClusterMax = 8;

template <typename T, int DPAD, int ROWWARPS>
struct Geom {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int TK = F32 ? 32 : 64;  // states a tile
    static constexpr int KEYWARPS = kWarps / ROWWARPS;
    static constexpr int NK = TK / KEYWARPS;  // states a warp and tile
    static constexpr int ROWS = 16 * ROWWARPS;
    static constexpr int CTAS = F32 && DPAD == 32 ? 4 : 2;  // an SM: registers are given up for them (fp32, d = 32: 58 -> 50 us)
    static constexpr int UNIT = 16 / sizeof(T);  // elements of 16 bytes
    static constexpr int LD = DPAD + UNIT;       // row pitch in shared memory: 16 bytes more, no bank conflicts
    static constexpr int STAGES = ROWWARPS == 1 ? 3 : 2;
    static constexpr int TILE = TK * LD;  // elements
    static constexpr int Q_BYTES = ROWS * LD * static_cast<int>(sizeof(T));
    static constexpr int RING_BYTES = STAGES * 2 * TILE * static_cast<int>(sizeof(T));
    // After the loop the ring's memory holds the warps' sums: [KEYWARPS][ROWS][DPAD] floats.
    static constexpr int SUM_BYTES = KEYWARPS * ROWS * DPAD * 4;
    static constexpr int OFF_RING = Q_BYTES;
    static constexpr int OFF_STATS = OFF_RING + (RING_BYTES > SUM_BYTES ? RING_BYTES : SUM_BYTES);
    // m, l of [kWarps][16]; joined m, l of [ROWS]; weights of [kClusterMax][ROWS]
    static constexpr int BYTES = OFF_STATS + 4 * (2 * kWarps * 16 + 2 * ROWS + kClusterMax * ROWS);
};

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank)
{
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

struct SplitArgs {
    AttnArgs a;
    int rows;        // N group packed rows a key head
    int row_blocks;  // CTAs of ROWS of them
    int splits;      // of the states
    int cluster;     // the splits form a cluster
    float* part_o;   // workspace: (B Hkv rows, splits, d) sums, when splits > 1 without a cluster
    float2* part_ml; // (B Hkv rows, splits) maximum and denominator
};

// out, out_lo and lse of packed row r of (b, hk), feature f.
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int b, int hk, int64_t r, int f, float v)
{
    const int64_t n = r / a.group;
    const int h = hk * a.group + static_cast<int>(r % a.group);
    const int64_t at = ((static_cast<int64_t>(b) * a.N + n) * a.Hq + h) * a.d + f;
    const T y = from_f<T>(v);
    static_cast<T*>(a.out)[at] = y;
    if (a.out_lo) static_cast<T*>(a.out_lo)[at] = from_f<T>((v - to_f(y)) * kLoScale<T>);
}
__device__ __forceinline__ void store_lse(const AttnArgs& a, int b, int hk, int64_t r, float v)
{
    if (!a.lse) return;
    const int64_t n = r / a.group;
    const int h = hk * a.group + static_cast<int>(r % a.group);
    a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.N + n] = v;
}
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.f : ex2f(m - top); }

template <typename T, int DPAD, int ROWWARPS, int VB>
__global__ void __launch_bounds__(kThreads, Geom<T, DPAD, ROWWARPS>::CTAS) attend_split_kernel(const __grid_constant__ SplitArgs f)
{
    using G = Geom<T, DPAD, ROWWARPS>;
    constexpr int UPR = DPAD / G::UNIT;          // 16-byte units a row
    const AttnArgs& a = f.a;
    extern __shared__ __align__(128) unsigned char sm[];
    T* sq = reinterpret_cast<T*>(sm);
    T* ring = reinterpret_cast<T*>(sm + G::OFF_RING);
    float* sums = reinterpret_cast<float*>(sm + G::OFF_RING);
    float* stat_m = reinterpret_cast<float*>(sm + G::OFF_STATS);
    float* stat_l = stat_m + kWarps * 16;
    float* row_m = stat_l + kWarps * 16;
    float* row_l = row_m + G::ROWS;
    float* weights = row_l + G::ROWS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rw = warp % ROWWARPS, kw = warp / ROWWARPS;

    const int split = static_cast<int>(blockIdx.x % f.splits);
    const int64_t unit = blockIdx.x / f.splits;
    const int rb = static_cast<int>(unit % f.row_blocks);
    const int hk = static_cast<int>(unit / f.row_blocks % a.Hkv), b = static_cast<int>(unit / f.row_blocks / a.Hkv);
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);
    if (!good && tid == 0) atomicOr(a.err, kErrBadLength);
    const int64_t r0 = static_cast<int64_t>(rb) * G::ROWS;
    const int64_t r1 = r0 + G::ROWS < f.rows ? r0 + G::ROWS : f.rows;

    // States that any row of this CTA touches, and this split's tiles of them.
    int64_t j0 = 0, j1 = 0;
    {
        const int64_t n0 = r0 / a.group, n1 = (r1 - 1) / a.group < nx - 1 ? (r1 - 1) / a.group : nx - 1;
        if (ny > 0 && n0 <= n1) {
            int64_t dummy;
            row_cells(a, n0, nx, ny, j0, dummy);
            row_cells(a, n1, nx, ny, dummy, j1);
        }
    }
    const int tiles = static_cast<int>((j1 - j0 + G::TK - 1) / G::TK);
    const int per = (tiles + f.splits - 1) / f.splits;
    const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;

    // The two rows of this thread (of its warp's 16) and their intervals.
    const int64_t ra = r0 + rw * 16 + (lane >> 2), rc = ra + 8;
    int64_t lo[2] = {0, 0}, hi[2] = {0, 0};
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int64_t r = x ? rc : ra, n = r / a.group;
        if (r < r1 && n < nx && ny > 0) row_cells(a, n, nx, ny, lo[x], hi[x]);
    }

    const T* kb = static_cast<const T*>(a.k) + b * a.ks.b + hk * a.ks.h;
    const T* vb = static_cast<const T*>(a.v) + b * a.vs.b + hk * a.vs.h;
    const auto load_tile = [&](int t) {
        T* kd = ring + (t - t0) % G::STAGES * 2 * G::TILE;
        const int64_t j = j0 + static_cast<int64_t>(t) * G::TK;
        const int u = tid % UPR;
        if (u * G::UNIT < a.d)
#pragma unroll
            for (int r = tid / UPR; r < G::TK; r += kThreads / UPR) {
                const bool on = j + r < ny;
                const int64_t row = on ? j + r : j0;
                copy_unit<T, VB>(kd + r * G::LD + u * G::UNIT, kb + row * a.ks.n + u * G::UNIT, u * G::UNIT, a.d, on);
                copy_unit<T, VB>(kd + G::TILE + r * G::LD + u * G::UNIT, vb + row * a.vs.n + u * G::UNIT, u * G::UNIT, a.d, on);
            }
    };
    // Features from d to DPAD are zero in every buffer.
    if (a.d < DPAD) {
        const int tail = DPAD - a.d;
        for (int e = tid; e < (G::ROWS + G::STAGES * 2 * G::TK) * tail; e += kThreads) {
            const int r = e / tail, c = a.d + e % tail;
            (r < G::ROWS ? sq + r * G::LD : ring + (r - G::ROWS) * G::LD)[c] = from_f<T>(0.f);
        }
    }
    {
        const int u = tid % UPR;
        if (u * G::UNIT < a.d)
            for (int r = tid / UPR; r < G::ROWS; r += kThreads / UPR) {
                const int64_t pr = r0 + r;
                const bool on = pr < r1;
                const int64_t n = on ? pr / a.group : 0;
                const int h = hk * a.group + static_cast<int>(on ? pr % a.group : 0);
                const T* src = static_cast<const T*>(a.q) + b * a.qs.b + n * a.qs.n + h * a.qs.h + u * G::UNIT;
                copy_unit<T, VB>(sq + r * G::LD + u * G::UNIT, src, u * G::UNIT, a.d, on);
            }
    }
#pragma unroll
    for (int s = 0; s < G::STAGES - 1; ++s) {
        if (t0 + s < t1) load_tile(t0 + s);
        cp_async_commit();
    }

    float o[DPAD / 8][4];
#pragma unroll
    for (int x = 0; x < DPAD / 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int t = t0; t < t1; ++t) {
        cp_async_wait<G::STAGES - 2>();
        __syncthreads();
        if (t + G::STAGES - 1 < t1) load_tile(t + G::STAGES - 1);
        cp_async_commit();
        const T* kt = ring + (t - t0) % G::STAGES * 2 * G::TILE + kw * G::NK * G::LD;
        const T* vt = kt + G::TILE;
        const int64_t jw = j0 + static_cast<int64_t>(t) * G::TK + kw * G::NK;  // this warp's first state
        // A warp passes over tiles without a cell of its rows (those of a band are not those of its CTA).
        const bool cells = (jw < hi[0] && jw + G::NK > lo[0]) || (jw < hi[1] && jw + G::NK > lo[1]);
        if (!__any_sync(kFull, cells)) continue;
        float s[G::NK / 8][4];
#pragma unroll
        for (int x = 0; x < G::NK / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[x][e] = 0.f;
        product_rows<T, DPAD, G::LD, G::NK / 8>(s, sq + rw * 16 * G::LD, kt, lane);
        // Scores in powers of two, masked; the row's maximum over the warp's states.
        const int64_t off0 = jw - lo[0], off1 = jw - lo[1];
        const bool inside = off0 >= 0 && off1 >= 0 && jw + G::NK <= hi[0] && jw + G::NK <= hi[1];
        const bool whole = __all_sync(kFull, inside);
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int x = 0; x < G::NK / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = s[x][e] * a.scale_log2;
                if (!whole) {
                    const int64_t j = jw + 8 * x + 2 * (lane & 3) + (e & 1);
                    if (j < lo[e >> 1] || j >= hi[e >> 1]) v = -INFINITY;
                }
                s[x][e] = v;
                top[e >> 1] = fmaxf(top[e >> 1], v);
            }
        float base[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(kFull, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(kFull, top[x], 2));
            const float fix = weight_of(m[x], top[x]);
            base[x] = top[x] == -INFINITY ? 0.f : top[x];
            m[x] = top[x];
            l[x] *= fix;
#pragma unroll
            for (int y = 0; y < DPAD / 8; ++y) {
                o[y][2 * x] *= fix;
                o[y][2 * x + 1] *= fix;
            }
        }
        // fp16 weights are kept 2^10 larger (a weight is at most one here): those down to 2^-24 of the warp's largest stay
        // normal numbers.
        constexpr float kShift = std::is_same<T, __half>::value ? 10.f : 0.f;
#pragma unroll
        for (int x = 0; x < G::NK / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[x][e] = ex2f(s[x][e] - base[e >> 1] + kShift);
                l[e >> 1] += s[x][e];
            }
        product_columns<T, DPAD, G::LD, G::NK / 8>(o, s, vt, lane);
    }
    cp_async_wait<0>();
    constexpr float kUnshift = std::is_same<T, __half>::value ? 0x1p-10f : 1.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(kFull, l[x], 1);
        l[x] += __shfl_xor_sync(kFull, l[x], 2);
        l[x] *= kUnshift;
        if ((lane & 3) == 0) {
            stat_m[warp * 16 + (lane >> 2) + 8 * x] = m[x];
            stat_l[warp * 16 + (lane >> 2) + 8 * x] = l[x];
        }
    }
    __syncthreads();  // every warp is done with the ring; its memory holds sums from here
    // Join the warps that share rows, in warp order.
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int row = (lane >> 2) + 8 * x;
        float top = -INFINITY, all = 0.f;
#pragma unroll
        for (int w = 0; w < G::KEYWARPS; ++w) top = fmaxf(top, stat_m[(w * ROWWARPS + rw) * 16 + row]);
#pragma unroll
        for (int w = 0; w < G::KEYWARPS; ++w)
            all += weight_of(stat_m[(w * ROWWARPS + rw) * 16 + row], top) * stat_l[(w * ROWWARPS + rw) * 16 + row];
        const float fix = weight_of(m[x], top) * kUnshift;
        float* to = sums + (static_cast<int64_t>(kw) * G::ROWS + rw * 16 + row) * DPAD + 2 * (lane & 3);
#pragma unroll
        for (int y = 0; y < DPAD / 8; ++y)
            *reinterpret_cast<float2*>(to + 8 * y) = make_float2(o[y][2 * x] * fix, o[y][2 * x + 1] * fix);
        if (kw == 0 && (lane & 3) == 0) {
            row_m[rw * 16 + row] = top;
            row_l[rw * 16 + row] = all;
        }
    }
    __syncthreads();
    const int rows = static_cast<int>(r1 - r0);
    const float nan = __int_as_float(0x7fc00000);
    if constexpr (G::KEYWARPS > 1) {
        for (int e = tid; e < rows * DPAD; e += kThreads) {
            float v = sums[e];
#pragma unroll
            for (int w = 1; w < G::KEYWARPS; ++w) v += sums[w * G::ROWS * DPAD + e];
            sums[e] = v;
        }
        __syncthreads();
    }
    if (f.splits == 1) {
        for (int e = tid; e < rows * DPAD; e += kThreads) {
            const int r = e / DPAD, c = e % DPAD;
            if (c >= a.d) continue;
            const float den = row_l[r];
            store_out<T>(a, b, hk, r0 + r, c, !good ? nan : (den > 0.f ? sums[e] / den : (den == 0.f ? 0.f : nan)));
        }
        for (int r = tid; r < rows; r += kThreads)
            store_lse(a, b, hk, r0 + r, row_m[r] == -INFINITY ? -INFINITY : row_m[r] + log2f(row_l[r]));
        return;
    }
    if (!f.cluster) {
        const int64_t head = (static_cast<int64_t>(b) * a.Hkv + hk) * f.rows + r0;
        for (int e = tid; e < rows * DPAD; e += kThreads) {
            const int r = e / DPAD, c = e % DPAD;
            if (c < a.d) f.part_o[((head + r) * f.splits + split) * a.d + c] = sums[e];
        }
        for (int r = tid; r < rows; r += kThreads)
            f.part_ml[(head + r) * f.splits + split] = make_float2(row_m[r], row_l[r]);
        return;
    }
    // The cluster's CTAs each finish a share of the rows' features from everyone's sums.
    cluster_sync();
    for (int r = tid; r < rows; r += kThreads) {
        float mm[kClusterMax], top = -INFINITY, all = 0.f;
#pragma unroll
        for (int c = 0; c < kClusterMax; ++c) {
            mm[c] = c < f.splits ? ld_cluster(row_m + r, c) : -INFINITY;
            top = fmaxf(top, mm[c]);
        }
#pragma unroll
        for (int c = 0; c < kClusterMax; ++c)
            if (c < f.splits) all += weight_of(mm[c], top) * ld_cluster(row_l + r, c);
        const float inv = !good ? nan : (all > 0.f ? 1.f / all : (all == 0.f ? 0.f : nan));
#pragma unroll
        for (int c = 0; c < kClusterMax; ++c) weights[c * G::ROWS + r] = weight_of(mm[c], top) * inv;
        if (split == 0) store_lse(a, b, hk, r0 + r, top == -INFINITY ? -INFINITY : top + log2f(all));
    }
    __syncthreads();
    for (int e = split * kThreads + tid; e < rows * DPAD; e += f.splits * kThreads) {
        const int r = e / DPAD, c = e % DPAD;
        if (c >= a.d) continue;
        float v = 0.f;
        for (int x = 0; x < f.splits; ++x) v = fmaf(weights[x * G::ROWS + r], ld_cluster(sums + e, x), v);
        store_out<T>(a, b, hk, r0 + r, c, good ? v : nan);
    }
    cluster_sync();  // no CTA ends while another reads its sums
}

// One warp a packed row: the splits' sums of the workspace, in split order.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_splits_kernel(const __grid_constant__ SplitArgs f)
{
    const AttnArgs& a = f.a;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (id >= static_cast<int64_t>(a.B) * a.Hkv * f.rows) return;
    const int64_t r = id % f.rows;
    const int hk = static_cast<int>(id / f.rows % a.Hkv), b = static_cast<int>(id / f.rows / a.Hkv);
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);
    const float2* ml = f.part_ml + id * f.splits;
    float top = -INFINITY, all = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < f.splits; ++s) top = fmaxf(top, ml[s].x);
    for (int s = 0; s < f.splits; ++s) {
        const float w = weight_of(ml[s].x, top);
        all += w * ml[s].y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 32 * e < a.d) v[e] = fmaf(w, f.part_o[(id * f.splits + s) * a.d + lane + 32 * e], v[e]);
    }
    const float inv = !good ? __int_as_float(0x7fc00000) : (all == 0.f ? 0.f : 1.f / all);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.d) store_out<T>(a, b, hk, r, lane + 32 * e, v[e] * inv);
    if (lane == 0) store_lse(a, b, hk, r, top == -INFINITY ? -INFINITY : top + log2f(all));
}

struct Plan {
    int row_warps, rows_per_cta, row_blocks, splits;
    bool cluster;
};

// How many ways the states are split: the number that keeps the SMs' two places for CTAs evenly filled, counting a
// split's fixed cost (launch, first tiles, joining) as three tiles. Measured at 16 x 1 x 32771 x 32/8 x 128 bf16.
Plan plan_of(const AttnArgs& a, bool f32)
{
    Plan p;
    const int64_t rows = a.N * a.group;
    p.row_warps = rows <= 16 ? 1 : 4;
    p.rows_per_cta = 16 * p.row_warps;
    p.row_blocks = static_cast<int>((rows + p.rows_per_cta - 1) / p.rows_per_cta);
    const int64_t units = static_cast<int64_t>(a.B) * a.Hkv * p.row_blocks;
    int dev = 0, sms = 0;
    if (current_sms(dev, sms) != cudaSuccess) sms = 148;
    const int64_t slots = 2 * sms;
    int64_t cells = a.M;
    if (a.bw >= 0 && a.N > 1) {  // what the rows of a CTA reach when the lengths are full
        const double slope = static_cast<double>(a.M) / static_cast<double>(a.N);
        const double reach = (2.0 * static_cast<double>(a.bw) + 1) * (slope > 1 ? 1 : slope) +
                             (static_cast<double>(p.rows_per_cta) / a.group + 1) * slope;
        if (reach < static_cast<double>(cells)) cells = static_cast<int64_t>(reach) + 1;
    }
    const int64_t tk = f32 ? 32 : 64, tiles = (cells + tk - 1) / tk;
    p.splits = 1;
    p.cluster = true;
    int64_t best = (units + slots - 1) / slots * (tiles + 3);
    for (int s = 2; s <= kClusterMax && s <= tiles; ++s) {
        const int64_t cost = (units * s + slots - 1) / slots * ((tiles + s - 1) / s + 3);
        if (cost < best) {
            best = cost;
            p.splits = s;
        }
    }
    const int64_t wide = slots / units < tiles / 8 ? slots / units : tiles / 8;
    if (wide >= 2 * kClusterMax) {
        p.splits = static_cast<int>(wide < 128 ? wide : 128);
        p.cluster = false;
    }
    return p;
}

template <typename T, int DPAD, int ROWWARPS, int VB>
cudaError_t launch(const SplitArgs& f, cudaStream_t s)
{
    using G = Geom<T, DPAD, ROWWARPS>;
    static_assert(G::CTAS * (G::BYTES + 1024) <= 228 * 1024, "the CTAs of an SM");
    const auto kernel = attend_split_kernel<T, DPAD, ROWWARPS, VB>;
    static std::atomic<bool> allowed[128];
    cudaError_t e = allow_smem(kernel, G::BYTES, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(f.a.B) * f.a.Hkv * f.row_blocks * f.splits));
    c.blockDim = dim3(kThreads);
    c.dynamicSmemBytes = G::BYTES;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = f.cluster ? static_cast<unsigned>(f.splits) : 1;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    e = cudaLaunchKernelEx(&c, kernel, f);
    if (e != cudaSuccess) return e;
    count_launch();
    if (f.splits > 1 && !f.cluster) {
        const int64_t rows = static_cast<int64_t>(f.a.B) * f.a.Hkv * f.rows;
        join_splits_kernel<T><<<static_cast<unsigned>((rows + kWarps - 1) / kWarps), kThreads, 0, s>>>(f);
        count_launch();
    }
    return cudaGetLastError();
}

template <typename T, int DPAD, int ROWWARPS>
cudaError_t launch_vb(const SplitArgs& f, int vb, cudaStream_t s)
{
    if (vb == 16) return launch<T, DPAD, ROWWARPS, 16>(f, s);
    if (vb >= 4) return launch<T, DPAD, ROWWARPS, 4>(f, s);
    if constexpr (sizeof(T) == 2) return launch<T, DPAD, ROWWARPS, 2>(f, s);
    return cudaErrorInvalidValue;
}

template <typename T, int ROWWARPS>
cudaError_t launch_d(const SplitArgs& f, int vb, cudaStream_t s)
{
    if (f.a.d <= 32) return launch_vb<T, 32, ROWWARPS>(f, vb, s);
    if (f.a.d <= 64) return launch_vb<T, 64, ROWWARPS>(f, vb, s);
    return launch_vb<T, 128, ROWWARPS>(f, vb, s);
}

template <typename T>
cudaError_t forward_t(SplitArgs& f, const Plan& p, cudaStream_t s)
{
    const AttnArgs& a = f.a;
    const int vb = copy_bytes(step_bits<T>(a.q, a.qs) | step_bits<T>(a.k, a.ks) | step_bits<T>(a.v, a.vs) | a.d * sizeof(T));
    return p.row_warps == 1 ? launch_d<T, 1>(f, vb, s) : launch_d<T, 4>(f, vb, s);
}

}  // namespace

size_t attention_split_workspace_bytes(const AttnArgs& a, int dtype)
{
    const Plan p = plan_of(a, dtype == SDTW_F32);
    if (p.cluster) return 0;
    return static_cast<size_t>(a.B) * a.Hkv * static_cast<size_t>(a.N * a.group) * p.splits * (a.d + 2) * sizeof(float);
}

cudaError_t attention_split_forward(const AttnArgs& a, int dtype, void* workspace, cudaStream_t s)
{
    const Plan p = plan_of(a, dtype == SDTW_F32);
    SplitArgs f{};
    f.a = a;
    f.rows = static_cast<int>(a.N * a.group);
    f.row_blocks = p.row_blocks;
    f.splits = p.splits;
    f.cluster = p.cluster;
    f.part_ml = static_cast<float2*>(workspace);
    f.part_o = static_cast<float*>(workspace) + 2 * static_cast<size_t>(a.B) * a.Hkv * f.rows * p.splits;
    if (dtype == SDTW_F32) return forward_t<float>(f, p, s);
    if (dtype == SDTW_F16) return forward_t<__half>(f, p, s);
    return forward_t<__nv_bfloat16>(f, p, s);
}

}  // namespace sdtw
