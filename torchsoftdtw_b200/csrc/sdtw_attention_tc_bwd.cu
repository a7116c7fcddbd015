// Gradients of cross attention of 16-bit operands on the tensor cores (tcgen05), in two launches without atomics on
// results: dq by tiles of queries, then dk and dv by tiles of states. Both form S and dP again:
//   P = 2^(s scale / ln 2 - lse),  dS = P (dP - delta),  delta = do . (o + o_lo)
//   dq = scale dS K;   dv = P^T dO,  dk = scale dS^T Q  (S^T = K Q^T and dP^T = V dO^T directly, states as rows)
// Seven products where one launch with atomic sums of dq would take five: the price of sums in one fixed order.
// P and dS go back over S and dP in tensor memory as the 16-bit A operand of the next product, so nothing of size
// queries x states leaves the SM. One warp issues all products, in an order in which the products that wait for the
// elementwise warps alternate with those that do not: in dk/dv  dV(i), S(i+1) | dK(i), dP(i+1), while the elementwise
// warps form dS(i) | P(i+1).
//
// fp16: P is kept 2^10 larger and dS scaled by a power of two that brings the rows' |do| to [8, 16) (a row's own in
// dq, where a row is a lane; the largest of the head in dk), so that neither under- nor overflows where the gradients do not.
#include <mutex>
#include <type_traits>

#include "sdtw_attention.h"
#include "sdtw_attention_tc.h"
#include "sdtw_tc.cuh"

namespace sdtw {

using namespace tc;

namespace {

constexpr int kTile = 128;  // rows of a product: queries in dq, states in dk/dv

template <typename T>
constexpr bool is_half = std::is_same<T, __half>::value;
template <typename T>
constexpr float kPShift = is_half<T> ? 10.f : 0.f;

struct BwdArgs {
    AttnArgs a;
    uint64_t timeout_ns;
    int tiles;        // CTAs a head
    int dn;           // d rounded up to 16
    uint32_t* peak;   // fp16: (B, Hkv) bits of the largest |do|^2 of the head's rows
};

// A power of two that brings `norm2` = |do|^2 to [64, 256), or one.
__device__ __forceinline__ float gradient_scale(float norm2)
{
    if (!(norm2 > 1e-30f) || !(norm2 < 1e30f)) return 1.f;
    return exp2f(3.f - floorf(0.5f * log2f(norm2)));
}

template <typename T, int DPAD>
struct DqGeom {
    static constexpr int KT = DPAD == 128 ? 128 : 64;  // states a tile
    static constexpr int WGS = KT / 64;                // elementwise warpgroups, 64 columns each
    static constexpr int ROW_BYTES = kTile * DPAD * 2; // Q, dO
    static constexpr int COL_BYTES = KT * DPAD * 2;    // K, V
    static constexpr int ROW_BLOCK = kTile * 128, COL_BLOCK = KT * 128;
    static constexpr int NBLOCK = DPAD / 64;
    static constexpr int STAGES = 2;
    static constexpr int OFF_DO = ROW_BYTES;
    static constexpr int OFF_RING = 2 * ROW_BYTES;  // STAGES of (K, V)
    static constexpr int OFF_STAT = OFF_RING + STAGES * 2 * COL_BYTES;  // delta, |do|^2 of the rows
    static constexpr int OFF_BAR = OFF_STAT + 2 * kTile * 4;
    // row_full, fix, k_full[S], k_empty[S], v_full[S], v_empty[S], s_full, s_free, dp_full, dp_free, ds_full, ds_free, acc
    static constexpr int NBAR = 2 + 4 * STAGES + 7;
    static constexpr int OFF_MISC = OFF_BAR + 8 * NBAR;
    static constexpr int BYTES = OFF_MISC + 32 + 1024;
    static constexpr uint32_t S_COL = 0, DP_COL = KT, DS_COL = 2 * KT, ACC_COL = 2 * KT + KT / 2;
    static constexpr uint32_t TMEM_COLS = ACC_COL + DPAD <= 256 ? 256 : 512;
    static constexpr int WARPS = 4 * WGS;
    static constexpr int THREADS = 32 * (WARPS + 2);
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

template <typename T, int DPAD>
__global__ void __launch_bounds__(DqGeom<T, DPAD>::THREADS, DPAD == 64 ? 2 : 1)
    attend_dq_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg,
                        const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                        const __grid_constant__ BwdArgs f)
{
    using G = DqGeom<T, DPAD>;
    const AttnArgs& a = f.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row_full = base + G::OFF_BAR, fix = row_full + 8, k_full = fix + 8, k_empty = k_full + 8 * G::STAGES;
    const uint32_t v_full = k_empty + 8 * G::STAGES, v_empty = v_full + 8 * G::STAGES, s_full = v_empty + 8 * G::STAGES;
    const uint32_t s_free = s_full + 8, dp_full = s_free + 8, dp_free = dp_full + 8, ds_full = dp_free + 8;
    const uint32_t ds_free = ds_full + 8, acc_full = ds_free + 8;
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC);
    float* s_delta = reinterpret_cast<float*>(sm + G::OFF_STAT);
    float* s_norm = s_delta + kTile;
    const Bound bound{f.timeout_ns, reinterpret_cast<volatile int*>(misc + 1), a.err};

    const int qt = static_cast<int>(blockIdx.x % f.tiles);
    const int h = static_cast<int>(blockIdx.x / f.tiles % a.Hq), b = static_cast<int>(blockIdx.x / f.tiles / a.Hq);
    const int hk = h / a.group;
    const int row0 = qt * kTile;
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);
    if (tid == 0) {
        mbar_init(row_full, 1);
        mbar_init(fix, 1);
        for (int s = 0; s < 4 * G::STAGES; ++s) mbar_init(k_full + 8 * s, 1);
        mbar_init(s_full, 1);
        mbar_init(s_free, G::WARPS);
        mbar_init(dp_full, 1);
        mbar_init(dp_free, G::WARPS);
        mbar_init(ds_full, G::WARPS);
        mbar_init(ds_free, 1);
        mbar_init(acc_full, 1);
        int first = 0, last = 0;
        if (row0 < nx && ny > 0) {
            int64_t lo, hi, lo1, hi1;
            row_cells(a, row0, nx, ny, lo, hi);
            row_cells(a, (row0 + kTile < nx ? row0 + kTile : nx) - 1, nx, ny, lo1, hi1);
            first = static_cast<int>(lo / G::KT);
            last = static_cast<int>((hi1 + G::KT - 1) / G::KT);
        }
        misc[2] = first;
        misc[3] = last;
        *bound.abort = 0;
        if (!good) atomicOr(a.err, kErrBadLength);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == G::WARPS) tmem_alloc(base + G::OFF_MISC, G::TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
    const int ja = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 2));
    const int jb = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 3));

    if (warp == G::WARPS + 1) {
        // ---------------- TMA ----------------
        int issued_k = 0, issued_v = 0, fixes = 0;
        bool ok = true;
        if (ja < jb) {
            if (lane == 0) {
                mbar_expect_tx(row_full, 2 * G::ROW_BYTES);
                for (int x = 0; x < G::NBLOCK; ++x) {
                    tma_load_4d(base + x * G::ROW_BLOCK, &mq, row_full, 64 * x, row0, h, b);
                    tma_load_4d(base + G::OFF_DO + x * G::ROW_BLOCK, &mg, row_full, 64 * x, row0, h, b);
                }
            }
            for (int j = ja; j < jb && ok; ++j) {
                const int n = j - ja, st = n % G::STAGES;
                const int64_t left = ny - static_cast<int64_t>(j) * G::KT;
                const bool clear = left < G::KT && ny < a.M;  // rows past the length may hold NaN
                for (int is_v = 0; is_v < 2 && ok; ++is_v) {
                    const uint32_t fullb = (is_v ? v_full : k_full) + 8 * st, emptyb = (is_v ? v_empty : k_empty) + 8 * st;
                    if (n >= G::STAGES && !mbar_wait(emptyb, (n / G::STAGES - 1) & 1, bound)) {
                        ok = false;
                        break;
                    }
                    const int at = G::OFF_RING + (2 * st + is_v) * G::COL_BYTES;
                    const uint32_t bar = clear ? fix : fullb;
                    if (lane == 0) {
                        mbar_expect_tx(bar, G::COL_BYTES);
                        for (int x = 0; x < G::NBLOCK; ++x)
                            tma_load_4d(base + at + x * G::COL_BLOCK, is_v ? &mv : &mk, bar, 64 * x, j * G::KT, hk, b);
                    }
                    __syncwarp();
                    if (clear) {
                        if (!mbar_wait(fix, fixes & 1, bound)) ok = false;
                        ++fixes;
                        for (int x = 0; x < G::NBLOCK; ++x)
                            for (int u = static_cast<int>(left) * 8 + lane; u < G::KT * 8; u += 32)
                                *reinterpret_cast<uint4*>(sm + at + x * G::COL_BLOCK + 16 * u) = make_uint4(0, 0, 0, 0);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(fullb);
                    }
                    ++(is_v ? issued_v : issued_k);
                }
            }
            mbar_drain(row_full, 0, f.timeout_ns);
            for (int n = issued_k < G::STAGES ? 0 : issued_k - G::STAGES; n < issued_k; ++n)
                mbar_drain(k_full + 8 * (n % G::STAGES), (n / G::STAGES) & 1, f.timeout_ns);
            for (int n = issued_v < G::STAGES ? 0 : issued_v - G::STAGES; n < issued_v; ++n)
                mbar_drain(v_full + 8 * (n % G::STAGES), (n / G::STAGES) & 1, f.timeout_ns);
        }
    } else if (warp == G::WARPS) {
        // ---------------- MMA ----------------
        if (ja < jb) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(G::KT, false), idesc_q = mma_idesc<T>(f.dn, true);
            const int n = jb - ja;
            const auto product = [&](uint32_t d, int rows_at, int cols_at) {
                const uint64_t rd = desc_k(base + rows_at), cd = desc_k(base + cols_at);
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k)  // features past d are zero; a branch between products costs more
                    mma_ss(tmem + d, desc_at(rd, (k / 4) * G::ROW_BLOCK + (k % 4) * 32),
                           desc_at(cd, (k / 4) * G::COL_BLOCK + (k % 4) * 32), idesc_s, k > 0, leader);
            };
            const auto k_at = [&](int i) { return G::OFF_RING + 2 * (i % G::STAGES) * G::COL_BYTES; };
            const auto scores = [&](int i) {
                if (!mbar_wait(k_full + 8 * (i % G::STAGES), (i / G::STAGES) & 1, bound)) return false;
                if (i > 0 && !mbar_wait(s_free, (i - 1) & 1, bound)) return false;
                fence_after();
                product(G::S_COL, 0, k_at(i));
                mma_commit(s_full, leader);
                return true;
            };
            const auto dprobs = [&](int i) {
                if (!mbar_wait(v_full + 8 * (i % G::STAGES), (i / G::STAGES) & 1, bound)) return false;
                if (i > 0 && !mbar_wait(dp_free, (i - 1) & 1, bound)) return false;
                fence_after();
                product(G::DP_COL, G::OFF_DO, k_at(i) + G::COL_BYTES);
                mma_commit(dp_full, leader);
                mma_commit(v_empty + 8 * (i % G::STAGES), leader);
                return true;
            };
            bool ok = mbar_wait(row_full, 0, bound) && scores(0) && dprobs(0);
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) ok = scores(i + 1) && dprobs(i + 1);
                ok = ok && mbar_wait(ds_full, i & 1, bound);
                if (!ok) break;
                fence_after();
                const uint64_t kd = desc_mn(base + k_at(i), G::COL_BLOCK);
#pragma unroll
                for (int k = 0; k < G::KT / 16; ++k)
                    mma_ts(tmem + G::ACC_COL, tmem + G::DS_COL + 8 * k, desc_at(kd, 2048 * k), idesc_q, i > 0 || k > 0, leader);
                mma_commit(ds_free, leader);
                mma_commit(k_empty + 8 * (i % G::STAGES), leader);
            }
            mma_commit(acc_full, leader);
            mbar_drain(acc_full, 0, f.timeout_ns);  // before the tensor memory is given back
        }
        __syncwarp();
    } else {
        // ---------------- elementwise: one row a thread, 64 columns a warpgroup ----------------
        // delta and |do|^2 of the tile's rows: LPR lanes a row.
        constexpr int LPR = DPAD / 8, RPW = 32 / LPR;
#pragma unroll 4
        for (int r0 = warp * RPW; r0 < kTile; r0 += G::WARPS * RPW) {
            const int r = r0 + lane / LPR, c = lane % LPR * 8;
            const int64_t i = row0 + r;
            float dot = 0.f, nrm = 0.f;
            if (i < nx && c < a.d && ny > 0) {
                const T* gp = static_cast<const T*>(a.dout) + b * a.gs.b + i * a.gs.n + h * a.gs.h + c;
                const int64_t at = ((static_cast<int64_t>(b) * a.N + i) * a.Hq + h) * a.d + c;
                const Vec<T, 8> g = *reinterpret_cast<const Vec<T, 8>*>(gp);
                const Vec<T, 8> o = *reinterpret_cast<const Vec<T, 8>*>(static_cast<const T*>(a.o) + at);
                Vec<T, 8> lo{};
                if (a.o_lo) lo = *reinterpret_cast<const Vec<T, 8>*>(static_cast<const T*>(a.o_lo) + at);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float gf = to_f(g.e[e]);
                    dot = fmaf(gf, to_f(o.e[e]) + to_f(lo.e[e]), dot);
                    nrm = fmaf(gf, gf, nrm);
                }
            }
#pragma unroll
            for (int x = LPR / 2; x > 0; x >>= 1) {
                dot += __shfl_xor_sync(kFull, dot, x);
                nrm += __shfl_xor_sync(kFull, nrm, x);
            }
            if (lane % LPR == 0) {
                s_delta[r] = dot;
                s_norm[r] = nrm;
                if (i < a.N) a.delta[(static_cast<int64_t>(b) * a.Hq + h) * a.N + i] = dot;
                if (is_half<T> && i < nx) atomicMax(f.peak + b * a.Hkv + hk, __float_as_uint(nrm));
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * G::WARPS) : "memory");
        const int wg = warp >> 2, r = tid & 127;
        const int64_t i = row0 + r;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + G::S_COL + 64 * wg, tdp = tmem + lanes + G::DP_COL + 64 * wg;
        const uint32_t tds = tmem + lanes + G::DS_COL + 32 * wg;
        int64_t lo = 0, hi = 0;
        if (i < nx && ny > 0) row_cells(a, i, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        const float lse = width > 0 ? a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.N + i] : INFINITY;
        const float gscale = is_half<T> ? gradient_scale(s_norm[r]) : 1.f;
        const float cf = is_half<T> ? gscale * exp2f(-kPShift<T>) : 1.f;
        const float delta = s_delta[r] * cf, bias = kPShift<T> - lse;
        bool ok = true;
        for (int j = ja; j < jb; ++j) {
            const int it = j - ja;
            if (!(ok = mbar_wait(s_full, it & 1, bound))) break;
            fence_after();
            uint32_t s[64], p[64];
            tmem_ld32(ts, s);
            tmem_ld32(ts + 32, s + 32);
            wait_ld();
            settle(s);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free);
            const int off = j * G::KT + 64 * wg - ilo;
            const bool whole = __all_sync(kFull, off >= 0 && off + 64 <= width);
#pragma unroll
            for (int c = 0; c < 64; ++c)
                s[c] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c]), a.scale_log2, bias)));
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0;
            }
            if (!(ok = mbar_wait(dp_full, it & 1, bound))) break;
            fence_after();
            tmem_ld32(tdp, p);
            tmem_ld32(tdp + 32, p + 32);
            wait_ld();
            settle(p);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dp_free);
            if (it > 0 && !(ok = mbar_wait(ds_free, (it - 1) & 1, bound))) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int x = c + 2 * e;
                    const float d0 = is_half<T> ? fmaf(__uint_as_float(p[x]), cf, -delta) : __uint_as_float(p[x]) - delta;
                    const float d1 = is_half<T> ? fmaf(__uint_as_float(p[x + 1]), cf, -delta) : __uint_as_float(p[x + 1]) - delta;
                    w[e] = pack2(__uint_as_float(s[x]) * d0, __uint_as_float(s[x + 1]) * d1, T());
                }
                tmem_st16(tds + c / 2, w);
            }
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full);
        }
        if (ok && jb > ja) ok = mbar_wait(acc_full, 0, bound);
        fence_after();
        ok = __all_sync(kFull, ok);
        const float back = a.scale / gscale;
        T* out = static_cast<T*>(a.dq) + ((static_cast<int64_t>(b) * a.N + i) * a.Hq + h) * a.d;
#pragma unroll
        for (int c = (DPAD / G::WGS) * wg; c < (DPAD / G::WGS) * (wg + 1); c += 16) {
            uint32_t o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0;
            if (c >= f.dn) break;
            if (jb > ja && ok) {
                tmem_ld16(tmem + lanes + G::ACC_COL + c, o);
                wait_ld();
                settle(o);
            }
            if (i >= a.N) continue;
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                if (c + e >= a.d) break;
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v0 = width > 0 ? __uint_as_float(o[e + 2 * x]) * back : 0.f;
                    float v1 = width > 0 ? __uint_as_float(o[e + 2 * x + 1]) * back : 0.f;
                    if (!ok) v0 = v1 = __int_as_float(0x7fc00000);
                    w[x] = pack2(v0, v1, T());
                }
                *reinterpret_cast<uint4*>(out + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        fence_before();
    }
    __syncthreads();
    if (warp == G::WARPS) {
        fence_after();
        tmem_free(tmem, G::TMEM_COLS);
    }
}

template <typename T, int DPAD>
struct DkvGeom {
    static constexpr int QT = DPAD == 128 ? 128 : 64;  // queries a tile
    static constexpr int WGS = QT / 64;
    static constexpr int ROW_BYTES = kTile * DPAD * 2;  // K, V
    static constexpr int COL_BYTES = QT * DPAD * 2;     // Q, dO
    static constexpr int ROW_BLOCK = kTile * 128, COL_BLOCK = QT * 128;
    static constexpr int NBLOCK = DPAD / 64;
    static constexpr int STAGES = 2;
    static constexpr int OFF_V = ROW_BYTES;
    static constexpr int OFF_RING = 2 * ROW_BYTES;  // STAGES of (Q, dO)
    static constexpr int OFF_STAT = OFF_RING + STAGES * 2 * COL_BYTES;  // STAGES of lse, delta of the tile's queries
    static constexpr int OFF_BAR = OFF_STAT + STAGES * 2 * QT * 4;
    // row_full, fix, q_full[S], q_empty[S], g_full[S], g_empty[S], s_full, p_full, dp_full, ds_full, acc
    static constexpr int NBAR = 2 + 4 * STAGES + 5;
    static constexpr int OFF_MISC = OFF_BAR + 8 * NBAR;
    static constexpr int BYTES = OFF_MISC + 32 + 1024;
    static constexpr uint32_t S_COL = 0, DP_COL = QT, DV_COL = 2 * QT, DK_COL = 2 * QT + DPAD;
    static constexpr uint32_t TMEM_COLS = DK_COL + DPAD <= 256 ? 256 : 512;
    static constexpr int WARPS = 4 * WGS;
    static constexpr int THREADS = 32 * (WARPS + 2);
    static_assert(BYTES <= 227 * 1024, "shared memory");
    static_assert(DK_COL + DPAD <= 512, "tensor memory");
};

template <typename T, int DPAD>
__global__ void __launch_bounds__(DkvGeom<T, DPAD>::THREADS, DPAD == 64 ? 2 : 1)
    attend_dkdv_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                          const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg,
                          const __grid_constant__ BwdArgs f)
{
    using G = DkvGeom<T, DPAD>;
    const AttnArgs& a = f.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row_full = base + G::OFF_BAR, fix = row_full + 8, q_full = fix + 8, q_empty = q_full + 8 * G::STAGES;
    const uint32_t g_full = q_empty + 8 * G::STAGES, g_empty = g_full + 8 * G::STAGES, s_full = g_empty + 8 * G::STAGES;
    const uint32_t p_full = s_full + 8, dp_full = p_full + 8, ds_full = dp_full + 8, acc_full = ds_full + 8;
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC);
    float* stats = reinterpret_cast<float*>(sm + G::OFF_STAT);
    const Bound bound{f.timeout_ns, reinterpret_cast<volatile int*>(misc + 1), a.err};

    const int kt = static_cast<int>(blockIdx.x % f.tiles);
    const int hk = static_cast<int>(blockIdx.x / f.tiles % a.Hkv), b = static_cast<int>(blockIdx.x / f.tiles / a.Hkv);
    const int row0 = kt * kTile;
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);
    if (tid == 0) {
        mbar_init(row_full, 1);
        mbar_init(fix, 1);
        for (int s = 0; s < 4 * G::STAGES; ++s) mbar_init(q_full + 8 * s, 1);
        mbar_init(s_full, 1);
        mbar_init(p_full, G::WARPS);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, G::WARPS);
        mbar_init(acc_full, 1);
        int first = 0, last = 0;
        if (row0 < ny && nx > 0) {
            int64_t lo, hi, lo1, hi1;
            column_cells(a, row0, nx, ny, lo, hi);
            column_cells(a, (row0 + kTile < ny ? row0 + kTile : ny) - 1, nx, ny, lo1, hi1);
            first = static_cast<int>(lo / G::QT);
            last = static_cast<int>((hi1 + G::QT - 1) / G::QT);
        }
        misc[2] = first;
        misc[3] = last;
        *bound.abort = 0;
        if (!good) atomicOr(a.err, kErrBadLength);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == G::WARPS) tmem_alloc(base + G::OFF_MISC, G::TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
    const int ia = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 2));
    const int nq = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 3)) - ia;  // tiles a query head
    const int n = nq > 0 ? nq * a.group : 0;
    // One power of two for all rows that share the sums.
    const float gscale = is_half<T> ? gradient_scale(__uint_as_float(f.peak[b * a.Hkv + hk])) : 1.f;
    const float cf = is_half<T> ? gscale * exp2f(-kPShift<T>) : 1.f;

    if (warp == G::WARPS + 1) {
        // ---------------- TMA, and the queries' statistics ----------------
        int issued_q = 0, issued_g = 0, fixes = 0;
        bool ok = true;
        if (n > 0) {
            if (lane == 0) {
                mbar_expect_tx(row_full, 2 * G::ROW_BYTES);
                for (int x = 0; x < G::NBLOCK; ++x) {
                    tma_load_4d(base + x * G::ROW_BLOCK, &mk, row_full, 64 * x, row0, hk, b);
                    tma_load_4d(base + G::OFF_V + x * G::ROW_BLOCK, &mv, row_full, 64 * x, row0, hk, b);
                }
            }
            for (int it = 0; it < n && ok; ++it) {
                const int st = it % G::STAGES, h = hk * a.group + it / nq, i0 = (ia + it % nq) * G::QT;
                const int64_t left = nx - i0;
                const bool clear = left < G::QT && nx < a.N;  // rows past the length may hold NaN
                for (int is_g = 0; is_g < 2 && ok; ++is_g) {
                    const uint32_t fullb = (is_g ? g_full : q_full) + 8 * st, emptyb = (is_g ? g_empty : q_empty) + 8 * st;
                    if (it >= G::STAGES && !mbar_wait(emptyb, (it / G::STAGES - 1) & 1, bound)) {
                        ok = false;
                        break;
                    }
                    if (!is_g) {
                        // A query past the length has P = 2^-inf = 0.
                        const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.N + i0;
#pragma unroll
                        for (int c = 0; c < G::QT; c += 32) {
                            const bool on = c + lane < left;
                            stats[st * 2 * G::QT + c + lane] = on ? kPShift<T> - a.lse[at + c + lane] : -INFINITY;
                            stats[st * 2 * G::QT + G::QT + c + lane] = on ? a.delta[at + c + lane] * cf : 0.f;
                        }
                        __syncwarp();
                    }
                    const int at = G::OFF_RING + (2 * st + is_g) * G::COL_BYTES;
                    const uint32_t bar = clear ? fix : fullb;
                    if (lane == 0) {
                        mbar_expect_tx(bar, G::COL_BYTES);
                        for (int x = 0; x < G::NBLOCK; ++x)
                            tma_load_4d(base + at + x * G::COL_BLOCK, is_g ? &mg : &mq, bar, 64 * x, i0, h, b);
                    }
                    __syncwarp();
                    if (clear) {
                        if (!mbar_wait(fix, fixes & 1, bound)) ok = false;
                        ++fixes;
                        for (int x = 0; x < G::NBLOCK; ++x)
                            for (int u = static_cast<int>(left) * 8 + lane; u < G::QT * 8; u += 32)
                                *reinterpret_cast<uint4*>(sm + at + x * G::COL_BLOCK + 16 * u) = make_uint4(0, 0, 0, 0);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(fullb);
                    }
                    ++(is_g ? issued_g : issued_q);
                }
            }
            mbar_drain(row_full, 0, f.timeout_ns);
            for (int x = issued_q < G::STAGES ? 0 : issued_q - G::STAGES; x < issued_q; ++x)
                mbar_drain(q_full + 8 * (x % G::STAGES), (x / G::STAGES) & 1, f.timeout_ns);
            for (int x = issued_g < G::STAGES ? 0 : issued_g - G::STAGES; x < issued_g; ++x)
                mbar_drain(g_full + 8 * (x % G::STAGES), (x / G::STAGES) & 1, f.timeout_ns);
        }
    } else if (warp == G::WARPS) {
        // ---------------- MMA ----------------
        if (n > 0) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(G::QT, false), idesc_o = mma_idesc<T>(f.dn, true);
            const auto product = [&](uint32_t d, int rows_at, int cols_at) {
                const uint64_t rd = desc_k(base + rows_at), cd = desc_k(base + cols_at);
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k)  // features past d are zero; a branch between products costs more
                    mma_ss(tmem + d, desc_at(rd, (k / 4) * G::ROW_BLOCK + (k % 4) * 32),
                           desc_at(cd, (k / 4) * G::COL_BLOCK + (k % 4) * 32), idesc_s, k > 0, leader);
            };
            // 64 columns of P or dS lie packed in the first 32 columns of their warpgroup's 64.
            const auto gradient = [&](uint32_t d, uint32_t src, int cols_at, bool more) {
                const uint64_t cd = desc_mn(base + cols_at, G::COL_BLOCK);
#pragma unroll
                for (int k = 0; k < G::QT / 16; ++k)
                    mma_ts(tmem + d, tmem + src + (k / 4) * 64 + (k % 4) * 8, desc_at(cd, 2048 * k), idesc_o, more || k > 0, leader);
            };
            const auto q_at = [&](int i) { return G::OFF_RING + 2 * (i % G::STAGES) * G::COL_BYTES; };
            const auto scores = [&](int i) {
                if (!mbar_wait(q_full + 8 * (i % G::STAGES), (i / G::STAGES) & 1, bound)) return false;
                fence_after();
                product(G::S_COL, 0, q_at(i));
                mma_commit(s_full, leader);
                return true;
            };
            const auto dprobs = [&](int i) {
                if (!mbar_wait(g_full + 8 * (i % G::STAGES), (i / G::STAGES) & 1, bound)) return false;
                fence_after();
                product(G::DP_COL, G::OFF_V, q_at(i) + G::COL_BYTES);
                mma_commit(dp_full, leader);
                return true;
            };
            bool ok = mbar_wait(row_full, 0, bound) && scores(0) && dprobs(0);
            for (int i = 0; ok && i < n; ++i) {
                ok = mbar_wait(p_full, i & 1, bound);
                if (!ok) break;
                fence_after();
                gradient(G::DV_COL, G::S_COL, q_at(i) + G::COL_BYTES, i > 0);
                mma_commit(g_empty + 8 * (i % G::STAGES), leader);
                if (i + 1 < n && !(ok = scores(i + 1))) break;
                ok = mbar_wait(ds_full, i & 1, bound);
                if (!ok) break;
                fence_after();
                gradient(G::DK_COL, G::DP_COL, q_at(i), i > 0);
                mma_commit(q_empty + 8 * (i % G::STAGES), leader);
                if (i + 1 < n) ok = dprobs(i + 1);
            }
            mma_commit(acc_full, leader);
            mbar_drain(acc_full, 0, f.timeout_ns);  // before the tensor memory is given back
        }
        __syncwarp();
    } else {
        // ---------------- elementwise: one state a thread, 64 queries a warpgroup ----------------
        const int wg = warp >> 2;
        const int64_t j = row0 + (tid & 127);
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + G::S_COL + 64 * wg, tdp = tmem + lanes + G::DP_COL + 64 * wg;
        int64_t lo = 0, hi = 0;
        if (j < ny && nx > 0) column_cells(a, j, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        bool ok = true;
        for (int it = 0; it < n; ++it) {
            const int st = it % G::STAGES;
            if (!(ok = mbar_wait(q_full + 8 * st, (it / G::STAGES) & 1, bound) && mbar_wait(s_full, it & 1, bound))) break;
            fence_after();
            const float* lse = stats + st * 2 * G::QT + 64 * wg;
            const float* delta = lse + G::QT;
            uint32_t s[64], p[64];
            tmem_ld32(ts, s);
            tmem_ld32(ts + 32, s + 32);
            wait_ld();
            settle(s);
            const int off = (ia + it % nq) * G::QT + 64 * wg - ilo;
            const bool whole = __all_sync(kFull, off >= 0 && off + 64 <= width);
#pragma unroll
            for (int c = 0; c < 64; c += 4) {
                const float4 b4 = *reinterpret_cast<const float4*>(lse + c);
                s[c] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c]), a.scale_log2, b4.x)));
                s[c + 1] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 1]), a.scale_log2, b4.y)));
                s[c + 2] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 2]), a.scale_log2, b4.z)));
                s[c + 3] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 3]), a.scale_log2, b4.w)));
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0;
            }
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = pack2(__uint_as_float(s[c + 2 * e]), __uint_as_float(s[c + 2 * e + 1]), T());
                tmem_st16(ts + c / 2, w);
            }
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
            if (!(ok = mbar_wait(dp_full, it & 1, bound))) break;
            fence_after();
            tmem_ld32(tdp, p);
            tmem_ld32(tdp + 32, p + 32);
            wait_ld();
            settle(p);
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int x = c + 2 * e;
                    const float4 d4 = *reinterpret_cast<const float4*>(delta + x);
                    const float dd[4] = {d4.x, d4.y, d4.z, d4.w};
                    float v[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float dp = __uint_as_float(p[x + y]);
                        v[y] = __uint_as_float(s[x + y]) * (is_half<T> ? fmaf(dp, cf, -dd[y]) : dp - dd[y]);
                    }
                    w[e] = pack2(v[0], v[1], T());
                    w[e + 1] = pack2(v[2], v[3], T());
                }
                tmem_st16(tdp + c / 2, w);
            }
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full);
        }
        if (ok && n > 0) ok = mbar_wait(acc_full, 0, bound);
        fence_after();
        ok = __all_sync(kFull, ok);
        const float back_k = a.scale / gscale, back_v = is_half<T> ? exp2f(-kPShift<T>) : 1.f;
        const int64_t at = ((static_cast<int64_t>(b) * a.M + j) * a.Hkv + hk) * a.d;
        for (int u = wg; u < 2 * (f.dn / 16); u += G::WGS) {  // 16 features of dv or dk at a time
            const bool is_k = u >= f.dn / 16;
            const int c = (is_k ? u - f.dn / 16 : u) * 16;
            const float back = is_k ? back_k : back_v;
            uint32_t o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0;
            if (n > 0 && ok) {
                tmem_ld16(tmem + lanes + (is_k ? G::DK_COL : G::DV_COL) + c, o);
                wait_ld();
                settle(o);
            }
            if (j >= a.M) continue;
            T* out = static_cast<T*>(is_k ? a.dk : a.dv) + at + c;
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                if (c + e >= a.d) break;
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v0 = width > 0 ? __uint_as_float(o[e + 2 * x]) * back : 0.f;
                    float v1 = width > 0 ? __uint_as_float(o[e + 2 * x + 1]) * back : 0.f;
                    if (!ok) v0 = v1 = __int_as_float(0x7fc00000);
                    w[x] = pack2(v0, v1, T());
                }
                *reinterpret_cast<uint4*>(out + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        fence_before();
    }
    __syncthreads();
    if (warp == G::WARPS) {
        fence_after();
        tmem_free(tmem, G::TMEM_COLS);
    }
}

template <typename K>
cudaError_t allow_smem(K kernel, int bytes)
{
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int DPAD>
cudaError_t backward_d(BwdArgs& f, cudaStream_t s)
{
    using GQ = DqGeom<T, DPAD>;
    using GK = DkvGeom<T, DPAD>;
    const AttnArgs& a = f.a;
    static_assert(GQ::KT == GK::QT, "one set of maps serves both launches");
    constexpr bool half = is_half<T>;
    // As rows of a product (128 a tile) and as columns (KT a tile).
    CUtensorMap q_rows, g_rows, k_cols, v_cols, k_rows, v_rows, q_cols, g_cols;
    const cudaError_t bad = cudaErrorInvalidValue;
    cudaError_t e;
    if (a.N > 0 && a.M > 0) {
        if (!attention_tile_map(&q_rows, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, kTile) ||
            !attention_tile_map(&g_rows, half, a.dout, a.gs, a.B, a.N, a.Hq, a.d, kTile) ||
            !attention_tile_map(&k_cols, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, GQ::KT) ||
            !attention_tile_map(&v_cols, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, GQ::KT) ||
            !attention_tile_map(&k_rows, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, kTile) ||
            !attention_tile_map(&v_rows, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, kTile) ||
            !attention_tile_map(&q_cols, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, GK::QT) ||
            !attention_tile_map(&g_cols, half, a.dout, a.gs, a.B, a.N, a.Hq, a.d, GK::QT))
            return bad;
    }
    if (half) {
        e = cudaMemsetAsync(f.peak, 0, sizeof(uint32_t) * static_cast<size_t>(a.B) * a.Hkv, s);
        if (e != cudaSuccess) return e;
    }
    if ((e = allow_smem(attend_dq_tc_kernel<T, DPAD>, GQ::BYTES)) != cudaSuccess) return e;
    if ((e = allow_smem(attend_dkdv_tc_kernel<T, DPAD>, GK::BYTES)) != cudaSuccess) return e;
    f.tiles = static_cast<int>((a.N + kTile - 1) / kTile);
    attend_dq_tc_kernel<T, DPAD><<<static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hq * f.tiles), GQ::THREADS, GQ::BYTES, s>>>(
        q_rows, g_rows, k_cols, v_cols, f);
    count_launch();
    f.tiles = static_cast<int>((a.M + kTile - 1) / kTile);
    attend_dkdv_tc_kernel<T, DPAD><<<static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hkv * f.tiles), GK::THREADS, GK::BYTES, s>>>(
        k_rows, v_rows, q_cols, g_cols, f);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t attention_tc_backward(const AttnArgs& a, bool bf16, uint32_t* peak, cudaStream_t s)
{
    BwdArgs f{};
    f.a = a;
    f.timeout_ns = static_cast<uint64_t>(wait_timeout_s() * 1e9);
    f.dn = (a.d + 15) / 16 * 16;
    f.peak = peak;
    if (bf16) return a.d <= 64 ? backward_d<__nv_bfloat16, 64>(f, s) : backward_d<__nv_bfloat16, 128>(f, s);
    return a.d <= 64 ? backward_d<__half, 64>(f, s) : backward_d<__half, 128>(f, s);
}

}  // namespace sdtw
