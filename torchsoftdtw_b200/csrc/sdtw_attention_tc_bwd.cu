// Gradients of cross attention of 16-bit operands on the tensor cores (tcgen05), in two launches without atomics on
// results: dq by tiles of queries, then dk and dv by tiles of states. Both form S and dP again:
//   P = 2^(s scale / ln 2 - lse),  dS = P (dP - delta),  delta = do . (o + o_lo)
//   dq = scale dS K;   dv = P^T dO,  dk = scale dS^T Q  (S^T = K Q^T and dP^T = V dO^T directly, states as rows)
// Seven products where one launch with atomic sums of dq would take five: the price of sums in one fixed order.
// P and dS go to tensor memory as the 16-bit A operand of the next product, so nothing of size queries x states leaves
// the SM. (Rounded once: gradients are off by 1.1 to 1.5 times their own rounding.) A CTA keeps 128 rows (of Q and dO, or of K and V) and streams 64 columns (of the other two) at a time; eight
// elementwise warps take a tile, two threads a row, 32 columns each. Products complete in no promised order among themselves,
// so whatever one of them reads is only overwritten when it has been awaited. To have work for the tensor core meanwhile, two
// tiles are in flight on an SM: of two CTAs (d <= 64), or of one that has two groups of elementwise warps and two sets of S and
// dP in tensor memory, for the even and the odd tiles (BUFS = 2).
//
// Bound, like the forward, by the elementwise step between products: 2 x 4096 x 4096 x 16 x 128 bf16 960 us (1000 TFLOP/s
// of the seven products; fp16 1007), 4 x 4096 x 4096 x 16 x 64 1060 us, 32 x 512 x 512 x 8 x 64 124 us (fp16 138), where the CTAs' first loads,
// of all SMs at once, take a third of the time. Sums of the tile before placed between S and dP: 10% slower.
//
// fp16: P is kept 2^14 larger and dS scaled by a power of two (a row's own in dq, where a row is a lane; one for the CTA's states in
// dk): sdtw_attention_range.cuh.
#include <mutex>
#include <type_traits>

#include "sdtw_attention_range.cuh"
#include "sdtw_attention_tc.h"
#include "sdtw_tc.cuh"

namespace sdtw {

using namespace tc;

namespace {

constexpr int kTile = 128;  // rows of a product: queries in dq, states in dk/dv

template <typename T>
constexpr bool is_half = std::is_same<T, __half>::value;
template <typename T>
constexpr float kPShift = is_half<T> ? kHalfShift : 0.f;
template <typename T>
constexpr float kPUnshift = is_half<T> ? kHalfUnshift : 1.f;

struct BwdArgs {
    AttnArgs a;
    uint64_t timeout_ns;
    int tiles;  // CTAs a head
    int dn;     // d rounded up to 16
    int stall;  // attention_stall()
};

constexpr int kCols = 64;  // columns of a product: states in dq, queries in dk/dv

// Shared memory: the two row operands, a ring of pairs of column tiles, statistics, barriers.
template <int DPAD>
struct Geom {
    static constexpr int ROW_BYTES = kTile * DPAD * 2, COL_BYTES = kCols * DPAD * 2;
    static constexpr int ROW_BLOCK = kTile * 128, COL_BLOCK = kCols * 128;  // 64 features of a tile
    static constexpr int NBLOCK = DPAD / 64;
    // Tiles in flight of the columns' first operand (K, or Q: scores run up to three tiles ahead of its last use) and second.
    static constexpr int S0 = DPAD == 128 ? 6 : 3, S1 = 3;
    static constexpr int BUFS = DPAD == 128 ? 2 : 1;  // tiles in flight
    static constexpr int ELEM_WARPS = 8 * BUFS, MMA_WARP = ELEM_WARPS, TMA_WARP = ELEM_WARPS + 1;
    static constexpr int THREADS = 32 * (ELEM_WARPS + 2);
    static constexpr int OFF_RING = 2 * ROW_BYTES;
    static constexpr int OFF_STAT = OFF_RING + (S0 + S1) * COL_BYTES;
    static constexpr int STAT_BYTES = 4 * (S0 * 2 * kCols > 2 * kTile ? S0 * 2 * kCols : 2 * kTile);
    static constexpr int OFF_BAR = OFF_STAT + STAT_BYTES;
    // row_full, fix, full[S0 + S1], empty[S0 + S1], acc_full, idle, and six a buffer
    static constexpr int NBAR = 4 + 2 * (S0 + S1) + 6 * BUFS;
    static_assert(S0 % BUFS == 0, "a group of elementwise warps sees every turn of its stages");
    static constexpr int OFF_MISC = OFF_BAR + 8 * NBAR;
    static constexpr int BYTES = OFF_MISC + 32 + 1024;
    static constexpr int CTAS = DPAD == 64 ? 2 : 1;  // an SM
    static_assert(CTAS * (BYTES + 1024) <= 228 * 1024, "shared memory");
};

// A place in the ring and the parity of its present turn.
template <int STAGES>
struct Turn {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next()
    {
        if (++at == STAGES) {
            at = 0;
            phase ^= 1;
        }
    }
};

// 32 rows of a warp pair's results, features 16 half, 16 half + 32, .. of each from tensor memory at `acc` (times `back`, zero
// where not `keep`), through shared memory (`rows`: 32 DPAD 16-bit values) to global rows `pitch` apart.
template <typename T, int DPAD>
__device__ __forceinline__ void store_rows(uint32_t acc, uint4* rows, int lane, int half, int pair, bool any, bool keep, bool broken,
                                           float back, int dn, int d, T* out, int64_t pitch, int64_t rows_left)
{
    constexpr int UPR = DPAD / 8;
    for (int c = 16 * half; c < dn; c += 32) {
        uint32_t o[16];
        if (any) {
            tmem_ld16(acc + c, o);
            wait_ld();
            settle(o);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            uint32_t v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float v0 = any && keep ? __uint_as_float(o[e + 2 * x]) * back : 0.f;
                float v1 = any && keep ? __uint_as_float(o[e + 2 * x + 1]) * back : 0.f;
                if (broken) v0 = v1 = __int_as_float(0x7fc00000);
                v[x] = pack2(v0, v1, T());
            }
            rows[lane * UPR + (((c + e) / 8) ^ (lane & 7))] = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
    asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair) : "memory");
#pragma unroll 4
    for (int r = half * (32 / UPR) + lane / UPR; r < 32; r += 2 * (32 / UPR))
        if (r < rows_left && lane % UPR * 8 < d)
            *reinterpret_cast<uint4*>(out + r * pitch + lane % UPR * 8) = rows[r * UPR + ((lane % UPR) ^ (r & 7))];
}

// The TMA warp's part: both row tiles, then pairs of column tiles in the order of use. Rows of a column tile past the length
// meet weights of zero but may hold NaN: the tile that the length ends in is cleared behind it before it is handed on.
// stats(stage, step) writes a tile's statistics before its first load.
template <int DPAD, typename COORDS, typename STATS>
__device__ __forceinline__ void load_tiles(unsigned char* sm, uint32_t base, const CUtensorMap* r1, const CUtensorMap* r2,
                                           const CUtensorMap* c1, const CUtensorMap* c2, int row0, int row_head, int b, int steps,
                                           int64_t length, int64_t extent, uint32_t row_full, uint32_t fix, uint32_t full,
                                           uint32_t empty, const Bound& bound, int lane, COORDS coords, STATS stats)
{
    using G = Geom<DPAD>;
    if (steps <= 0) return;
    if (lane == 0) {
        mbar_expect_tx(row_full, 2 * G::ROW_BYTES);
        for (int x = 0; x < G::NBLOCK; ++x) {
            tma_load_4d(base + x * G::ROW_BLOCK, r1, row_full, 64 * x, row0, row_head, b);
            tma_load_4d(base + G::ROW_BYTES + x * G::ROW_BLOCK, r2, row_full, 64 * x, row0, row_head, b);
        }
    }
    Turn<G::S0> turn0;
    Turn<G::S1> turn1;
    int issued[2] = {0, 0}, fixes = 0;
    bool ok = true;
    for (int t = 0; t < steps && ok; ++t) {
        int c0, head;
        coords(t, c0, head);
        const int64_t left = length - c0;
        const bool clear = left < kCols && length < extent;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int place = which ? G::S0 + turn1.at : turn0.at;
            const uint32_t fullb = full + 8 * place, emptyb = empty + 8 * place;
            ok = ok && (t < (which ? G::S1 : G::S0) || mbar_wait(emptyb, (which ? turn1.phase : turn0.phase) ^ 1, bound));
            if (!ok) break;
            if (which == 0) {
                stats(turn0.at, t);
                __syncwarp();
            }
            const int at = G::OFF_RING + place * G::COL_BYTES;
            const uint32_t bar = clear ? fix : fullb;
            if (lane == 0) {
                mbar_expect_tx(bar, G::COL_BYTES);
                for (int x = 0; x < G::NBLOCK; ++x)
                    tma_load_4d(base + at + x * G::COL_BLOCK, which ? c2 : c1, bar, 64 * x, c0, head, b);
            }
            __syncwarp();
            if (clear) {
                ok = mbar_wait(fix, fixes & 1, bound);
                if (!ok) mbar_drain(fix, fixes & 1, bound.timeout_ns);  // `full`, drained below, will not tell of this load
                ++fixes;
                for (int x = 0; x < G::NBLOCK; ++x)
                    for (int u = static_cast<int>(left) * 8 + lane; u < kCols * 8; u += 32)
                        *reinterpret_cast<uint4*>(sm + at + x * G::COL_BLOCK + 16 * u) = make_uint4(0, 0, 0, 0);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(fullb);
            }
            ++issued[which];
        }
        turn0.next();
        turn1.next();
    }
    // Every load has landed before the CTA ends (also after an abort).
    mbar_drain(row_full, 0, bound.timeout_ns);
    for (int t = issued[0] < G::S0 ? 0 : issued[0] - G::S0; t < issued[0]; ++t)
        mbar_drain(full + 8 * (t % G::S0), (t / G::S0) & 1, bound.timeout_ns);
    for (int t = issued[1] < G::S1 ? 0 : issued[1] - G::S1; t < issued[1]; ++t)
        mbar_drain(full + 8 * (G::S0 + t % G::S1), (t / G::S1) & 1, bound.timeout_ns);
}

// d = rows cols^T over all features (those past d are zero; a branch between products costs more than they do).
template <int DPAD>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t rows_at, uint32_t cols_at, uint32_t idesc, uint32_t leader)
{
    using G = Geom<DPAD>;
    const uint64_t rd = desc_k(rows_at), cd = desc_k(cols_at);
#pragma unroll
    for (int k = 0; k < DPAD / 16; ++k)
        mma_ss(d, desc_at(rd, (k / 4) * G::ROW_BLOCK + (k % 4) * 32), desc_at(cd, (k / 4) * G::COL_BLOCK + (k % 4) * 32), idesc,
               k > 0, leader);
}
// d += A cols, A the 128 x 64 operand at `a` in tensor memory: 32 columns of it packed in 16, `half` apart.
template <int DPAD>
__device__ __forceinline__ void mma_cols(uint32_t d, uint32_t a, uint32_t half, uint32_t cols_at, uint32_t idesc, bool more,
                                         uint32_t leader)
{
    using G = Geom<DPAD>;
    const uint64_t cd = desc_mn(cols_at, G::COL_BLOCK);
#pragma unroll
    for (int k = 0; k < kCols / 16; ++k)
        mma_ts(d, a + (k / 2) * half + (k % 2) * 8, desc_at(cd, 2048 * k), idesc, more || k > 0, leader);
}

// TAIL (d <= 32): what the rounding of dS dropped goes through a second product. With few features the scores' tails are heavier
// and a few large dS carry dq, whose rounding nothing averages: without it dq is off by 1.6 times its own rounding at
// d = 16 (1.4 from d = 64 on), with it by 1.1 times; 4 x 4096 x 4096 x 16 x 16 1.04 -> 1.16 ms. At d <= 32 tensor memory has room
// for it beside the narrow sum.
template <typename T, int DPAD, bool TAIL>
__global__ void __launch_bounds__(Geom<DPAD>::THREADS, Geom<DPAD>::CTAS)
    attend_dq_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg,
                        const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                        const __grid_constant__ BwdArgs f)
{
    using G = Geom<DPAD>;
    // Each buffer: S, dP, dS.
    constexpr uint32_t DP_COL = kCols, DS_COL = 2 * kCols, BUF_COLS = 2 * kCols + kCols / 2, ACC_COL = G::BUFS * BUF_COLS;
    constexpr uint32_t TAIL_COL = ACC_COL + DPAD, ALL_COLS = TAIL_COL + (TAIL ? kCols / 2 : 0);
    constexpr uint32_t TMEM_COLS = ALL_COLS <= 256 ? 256 : 512;
    static_assert(ALL_COLS <= 512 && (!TAIL || G::BUFS == 1), "tensor memory");
    const AttnArgs& a = f.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row_full = base + G::OFF_BAR, fix = row_full + 8, full = fix + 8, empty = full + 8 * (G::S0 + G::S1);
    const uint32_t acc_full = empty + 8 * (G::S0 + G::S1), idle = acc_full + 8, s_full = idle + 8, s_free = s_full + 8 * G::BUFS;
    const uint32_t dp_full = s_free + 8 * G::BUFS, dp_free = dp_full + 8 * G::BUFS, ds_full = dp_free + 8 * G::BUFS;
    const uint32_t ds_free = ds_full + 8 * G::BUFS;
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
        for (int s = 0; s < 2 * (G::S0 + G::S1); ++s) mbar_init(full + 8 * s, 1);
        mbar_init(acc_full, 1);
        mbar_init(idle, 1);
        for (int x = 0; x < G::BUFS; ++x) {
            mbar_init(s_full + 8 * x, 1);
            mbar_init(s_free + 8 * x, 8);
            mbar_init(dp_full + 8 * x, 1);
            mbar_init(dp_free + 8 * x, 8);
            mbar_init(ds_full + 8 * x, 8);
            mbar_init(ds_free + 8 * x, 1);
        }
        int first = 0, last = 0;
        if (row0 < nx && ny > 0) {
            int64_t lo, hi, lo1, hi1;
            row_cells(a, row0, nx, ny, lo, hi);
            row_cells(a, (row0 + kTile < nx ? row0 + kTile : nx) - 1, nx, ny, lo1, hi1);
            first = static_cast<int>(lo / kCols);
            last = static_cast<int>((hi1 + kCols - 1) / kCols);
        }
        misc[2] = first;
        misc[3] = last;
        *bound.abort = 0;
        if (!good) atomicOr(a.err, kErrBadLength);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == G::MMA_WARP) tmem_alloc(base + G::OFF_MISC, TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
    const int ja = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 2));
    const int n = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 3)) - ja;

    if (warp == G::TMA_WARP) {
        load_tiles<DPAD>(
            sm, base, &mq, &mg, &mk, &mv, row0, h, b, n, ny, a.M, row_full, fix, full, empty, bound, lane,
            [&](int t, int& c0, int& head) {
                c0 = (ja + t) * kCols;
                head = hk;
            },
            [](int, int) {});
    } else if (warp == G::MMA_WARP) {
        if (n > 0) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(kCols, false), idesc_q = mma_idesc<T>(f.dn, true);
            Turn<G::S0> now;
            const auto ring = [&](int at, int which) { return base + G::OFF_RING + ((which ? G::S0 : 0) + at) * G::COL_BYTES; };
            // S, and dP, of tile i, when the elementwise warps have read the last one of its buffer; then tile i's share of dq.
            Turn<G::S0> ks;
            Turn<G::S1> vs;
            const auto scores = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(full + 8 * ks.at, ks.phase, bound)) return false;
                if (i >= G::BUFS && !mbar_wait(s_free + 8 * x, (i / G::BUFS - 1) & 1, bound)) return false;
                fence_after();
                mma_rows<DPAD>(tmem + x * BUF_COLS, base, ring(ks.at, 0), idesc_s, leader);
                mma_commit(s_full + 8 * x, leader);
                ks.next();
                return true;
            };
            const auto dprobs = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(full + 8 * (G::S0 + vs.at), vs.phase, bound)) return false;
                if (i >= G::BUFS && !mbar_wait(dp_free + 8 * x, (i / G::BUFS - 1) & 1, bound)) return false;
                fence_after();
                mma_rows<DPAD>(tmem + x * BUF_COLS + DP_COL, base + G::ROW_BYTES, ring(vs.at, 1), idesc_s, leader);
                mma_commit(dp_full + 8 * x, leader);
                mma_commit(empty + 8 * (G::S0 + vs.at), leader);
                vs.next();
                return true;
            };
            const auto sums = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(ds_full + 8 * x, (i / G::BUFS) & 1, bound)) return false;
                fence_after();
                mma_cols<DPAD>(tmem + ACC_COL, tmem + x * BUF_COLS + DS_COL, 16, ring(now.at, 0), idesc_q, i > 0, leader);
                if constexpr (TAIL) mma_cols<DPAD>(tmem + ACC_COL, tmem + TAIL_COL, 16, ring(now.at, 0), idesc_q, true, leader);
                mma_commit(ds_free + 8 * x, leader);
                mma_commit(empty + 8 * now.at, leader);
                now.next();
                return true;
            };
            bool ok = mbar_wait(row_full, 0, bound);
            for (int i = 0; i < G::BUFS && i < n; ++i) ok = ok && scores(i) && dprobs(i);
            if (G::BUFS == 1) {
                for (int i = 0; ok && i < n; ++i) {
                    if (i + 1 < n) ok = scores(i + 1) && dprobs(i + 1);
                    ok = ok && sums(i);
                }
            } else {
                // (Sums of tile i - 1 between S and dP of the next: 10% slower, for the two groups then wait for each other.)
                for (int i = 0; ok && i < n; ++i) {
                    if (i + 2 < n) ok = scores(i + 2) && dprobs(i + 2);
                    ok = ok && sums(i);
                }
            }
            if (ok) mma_commit(acc_full, leader);  // else the elementwise warps' wait for it ends by the abort
            mma_commit(idle, leader);
            mbar_drain(idle, 0, f.timeout_ns);  // before the tensor memory is given back
        }
        __syncwarp();
    } else {
        // ---------------- elementwise: two threads a row, 32 columns each ----------------
        // delta and |do|^2 of the tile's rows: LPR lanes a row, all loads ahead of the sums (rows and features outside read a
        // place inside, and count as zero).
        constexpr int LPR = DPAD / 8, RPW = 32 / LPR, ROUNDS = kTile / (G::ELEM_WARPS * RPW);
        PeakPart v_part{};  // fp16: of the largest |v| of the tile's states
        if (n > 0) {
            if constexpr (is_half<T>) {
                const int64_t end = static_cast<int64_t>(ja + n) * kCols;
                v_part = value_part(a, b, hk, static_cast<int64_t>(ja) * kCols, end < ny ? end : ny);
            }
            Vec<T, 8> g[ROUNDS], o[ROUNDS], lo[ROUNDS];
            const int c = lane % LPR * 8 < a.d ? lane % LPR * 8 : 0;
#pragma unroll
            for (int t = 0; t < ROUNDS; ++t) {
                const int64_t i1 = row0 + (t * G::ELEM_WARPS + warp) * RPW + lane / LPR, i = i1 < nx ? i1 : row0;
                const int64_t at = ((static_cast<int64_t>(b) * a.N + i) * a.Hq + h) * a.d + c;
                g[t] = *reinterpret_cast<const Vec<T, 8>*>(static_cast<const T*>(a.dout) + b * a.gs.b + i * a.gs.n + h * a.gs.h + c);
                o[t] = *reinterpret_cast<const Vec<T, 8>*>(static_cast<const T*>(a.o) + at);
                lo[t] = a.o_lo ? *reinterpret_cast<const Vec<T, 8>*>(static_cast<const T*>(a.o_lo) + at) : Vec<T, 8>{};
            }
#pragma unroll
            for (int t = 0; t < ROUNDS; ++t) {
                const int r = (t * G::ELEM_WARPS + warp) * RPW + lane / LPR;
                const bool on = row0 + r < nx && lane % LPR * 8 < a.d;
                float dot = 0.f, nrm = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float gf = on ? to_f(g[t].e[e]) : 0.f;
                    dot = on ? fmaf(gf, fmaf(to_f(lo[t].e[e]), 1.f / kLoScale<T>, to_f(o[t].e[e])), dot) : 0.f;
                    nrm = fmaf(gf, gf, nrm);
                }
#pragma unroll
                for (int x = LPR / 2; x > 0; x >>= 1) {
                    dot += __shfl_xor_sync(kFull, dot, x);
                    nrm += __shfl_xor_sync(kFull, nrm, x);
                }
                if (lane % LPR == 0) {
                    s_delta[r] = dot;
                    s_norm[r] = nrm;
                    if (row0 + r < nx) a.delta[(static_cast<int64_t>(b) * a.Hq + h) * a.N + row0 + r] = dot;
                }
            }
        }
        const int x = warp >> 3, half = (warp >> 2) & 1, r = 32 * (warp & 3) + lane;  // x: the buffer of this group of warps
        const int64_t i = row0 + r;
        int64_t lo = 0, hi = 0;
        if (i < nx && ny > 0) row_cells(a, i, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        const float lse = width > 0 ? a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.N + i] : INFINITY;
        asm volatile("barrier.cta.sync 1, %0;" ::"n"(32 * G::ELEM_WARPS) : "memory");
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + x * BUF_COLS + 32 * half, tdp = ts + DP_COL;
        const uint32_t tds = tmem + lanes + x * BUF_COLS + DS_COL + 16 * half;
        float cf = 1.f;  // of dP and delta: the scale of dS, less the shift of P
        if (is_half<T> && n > 0) {
            if (warp < kTile / kPeakRows) {
                const int r1 = warp * kPeakRows + lane;
                const float norm2 = warp_maxf(fmaxf(s_norm[r1], s_norm[r1 + 32]));
                const float top = warp_maxf(fmaxf(fabsf(s_delta[r1]), fabsf(s_delta[r1 + 32])));
                if (lane == 0 && row0 + warp * kPeakRows < nx) raise_gradient_peak(a, b, hk, row0 + warp * kPeakRows, norm2, top);
            }
            cf = half_scale(fmaf(sqrtf(s_norm[r]), peak_of(v_part), fabsf(s_delta[r]))) * kHalfUnshift;
        }
        const float delta = s_delta[r] * cf, bias = kPShift<T> - lse;
        bool ok = true;
        for (int it = x; it < n; it += G::BUFS) {
            const uint32_t phase = (it / G::BUFS) & 1;
            if (!(ok = mbar_wait(s_full + 8 * x, phase, bound))) break;
            fence_after();
            uint32_t s[32], p[32];
            tmem_ld32(ts, s);
            wait_ld();
            settle(s);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + 8 * x);
            const int off = (ja + it) * kCols + 32 * half - ilo;
            const bool whole = __all_sync(kFull, off >= 0 && off + 32 <= width);
#pragma unroll
            for (int c = 0; c < 32; ++c)
                s[c] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c]), a.scale_log2, bias)));
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0;
            }
            if (!(ok = mbar_wait(dp_full + 8 * x, phase, bound))) break;
            fence_after();
            tmem_ld32(tdp, p);
            wait_ld();
            settle(p);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dp_free + 8 * x);
            uint32_t w[16], wt[TAIL ? 16 : 1];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p0 = __uint_as_float(p[2 * e]), p1 = __uint_as_float(p[2 * e + 1]);
                const float d0 = is_half<T> ? fmaf(p0, cf, -delta) : p0 - delta;
                const float d1 = is_half<T> ? fmaf(p1, cf, -delta) : p1 - delta;
                const float v0 = __uint_as_float(s[2 * e]) * d0, v1 = __uint_as_float(s[2 * e + 1]) * d1;
                w[e] = pack2(v0, v1, T());
                if constexpr (TAIL) {
                    const Vec<T, 2> head = *reinterpret_cast<const Vec<T, 2>*>(&w[e]);
                    wt[e] = pack2(v0 - to_f(head.e[0]), v1 - to_f(head.e[1]), T());
                }
            }
            if (it >= G::BUFS && !(ok = mbar_wait(ds_free + 8 * x, phase ^ 1, bound))) break;
            fence_after();
            tmem_st16(tds, w);
            if constexpr (TAIL) tmem_st16(tds + (TAIL_COL - DS_COL), wt);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0 && !(f.stall == 2 && blockIdx.x == 0 && warp == 0 && it == 0)) mbar_arrive(ds_full + 8 * x);
        }
        if (ok && n > 0) ok = mbar_wait(acc_full, 0, bound);
        fence_after();
        // Q's place holds the rows on their way out: all scores are done.
        const int64_t i0 = row0 + 32 * (warp & 3);
        if (x == 0)
            store_rows<T, DPAD>(tmem + lanes + ACC_COL, reinterpret_cast<uint4*>(sm) + (warp & 3) * 32 * (DPAD / 8), lane, half,
                            2 + (warp & 3), n > 0 && ok, width > 0, !ok, a.scale * kPUnshift<T> / cf, f.dn, a.d,
                            static_cast<T*>(a.dq) + ((static_cast<int64_t>(b) * a.N + i0) * a.Hq + h) * a.d,
                            static_cast<int64_t>(a.Hq) * a.d, a.N - i0);
        fence_before();
    }
    __syncthreads();
    if (warp == G::MMA_WARP) {
        fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
}

template <typename T, int DPAD>
__global__ void __launch_bounds__(Geom<DPAD>::THREADS, Geom<DPAD>::CTAS)
    attend_dkdv_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                          const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg,
                          const __grid_constant__ BwdArgs f)
{
    using G = Geom<DPAD>;
    // Each buffer: S, then P packed at the start of each half's columns; dP, then dS.
    constexpr uint32_t DP_COL = kCols, BUF_COLS = 2 * kCols, DV_COL = G::BUFS * BUF_COLS, DK_COL = DV_COL + DPAD;
    constexpr uint32_t TMEM_COLS = DK_COL + DPAD <= 256 ? 256 : 512;
    static_assert(DK_COL + DPAD <= 512, "tensor memory");
    const AttnArgs& a = f.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row_full = base + G::OFF_BAR, fix = row_full + 8, full = fix + 8, empty = full + 8 * (G::S0 + G::S1);
    const uint32_t acc_full = empty + 8 * (G::S0 + G::S1), idle = acc_full + 8, s_full = idle + 8, p_full = s_full + 8 * G::BUFS;
    const uint32_t dp_full = p_full + 8 * G::BUFS, ds_full = dp_full + 8 * G::BUFS, dv_done = ds_full + 8 * G::BUFS;
    const uint32_t dk_done = dv_done + 8 * G::BUFS;
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC);
    float* stats = reinterpret_cast<float*>(sm + G::OFF_STAT);  // S0 of (shift - lse, delta) of 64 queries
    const Bound bound{f.timeout_ns, reinterpret_cast<volatile int*>(misc + 1), a.err};

    const int kt = static_cast<int>(blockIdx.x % f.tiles);
    const int hk = static_cast<int>(blockIdx.x / f.tiles % a.Hkv), b = static_cast<int>(blockIdx.x / f.tiles / a.Hkv);
    const int row0 = kt * kTile;
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);
    if (tid == 0) {
        mbar_init(row_full, 1);
        mbar_init(fix, 1);
        for (int s = 0; s < 2 * (G::S0 + G::S1); ++s) mbar_init(full + 8 * s, 1);
        mbar_init(acc_full, 1);
        mbar_init(idle, 1);
        for (int x = 0; x < G::BUFS; ++x) {
            mbar_init(s_full + 8 * x, 1);
            mbar_init(p_full + 8 * x, 8);
            mbar_init(dp_full + 8 * x, 1);
            mbar_init(ds_full + 8 * x, 8);
            mbar_init(dv_done + 8 * x, 1);
            mbar_init(dk_done + 8 * x, 1);
        }
        int first = 0, last = 0;
        if (row0 < ny && nx > 0) {
            int64_t lo, hi, lo1, hi1;
            column_cells(a, row0, nx, ny, lo, hi);
            column_cells(a, (row0 + kTile < ny ? row0 + kTile : ny) - 1, nx, ny, lo1, hi1);
            first = static_cast<int>(lo / kCols);
            last = static_cast<int>((hi1 + kCols - 1) / kCols);
        }
        misc[2] = first;
        misc[3] = last;
        *bound.abort = 0;
        if (!good) atomicOr(a.err, kErrBadLength);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == G::MMA_WARP) tmem_alloc(base + G::OFF_MISC, TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
    const int ia = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 2));
    const int nq = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(misc + 3)) - ia;  // tiles a query head
    const int n = nq > 0 ? nq * a.group : 0;
    // fp16: one power of two for all rows that share the sums. (Formed by the warps apart, beside the first loads: 5% slower, for
    // the elementwise loop's registers.)
    float cf = 1.f;
    if (is_half<T> && n > 0) {
        const int64_t end = static_cast<int64_t>(ia + nq) * kCols;
        const float bound_s = gradient_bound(a, b, hk, static_cast<int64_t>(ia) * kCols, end < nx ? end : nx, row0,
                                             row0 + kTile < ny ? row0 + kTile : ny);
        cf = half_scale(bound_s) * kHalfUnshift;
    }

    if (warp == G::TMA_WARP) {
        int head = hk * a.group, tile = -1;  // of the step that coords() was last asked for
        load_tiles<DPAD>(
            sm, base, &mk, &mv, &mq, &mg, row0, hk, b, n, nx, a.N, row_full, fix, full, empty, bound, lane,
            [&](int, int& c0, int& hd) {
                if (++tile == nq) {
                    tile = 0;
                    ++head;
                }
                c0 = (ia + tile) * kCols;
                hd = head;
            },
            [&](int stage, int) {
                const int i0 = (ia + tile) * kCols;
                const int64_t at = (static_cast<int64_t>(b) * a.Hq + head) * a.N + i0;
                float* st = stats + stage * 2 * kCols;
#pragma unroll
                for (int c = lane; c < kCols; c += 32) {
                    const bool on = i0 + c < nx;  // a query past the length has P = 2^-inf = 0
                    st[c] = on ? kPShift<T> - a.lse[at + c] : -INFINITY;
                    st[kCols + c] = on ? a.delta[at + c] * cf : 0.f;
                }
            });
    } else if (warp == G::MMA_WARP) {
        if (n > 0) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(kCols, false), idesc_o = mma_idesc<T>(f.dn, true);
            Turn<G::S0> sq;  // the next S
            Turn<G::S1> sg;  // the next dP
            const auto ring = [&](int at, int which) { return base + G::OFF_RING + ((which ? G::S0 : 0) + at) * G::COL_BYTES; };
            // S (dP) of tile i, when the product that read P (dS) there has completed.
            const auto scores = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(full + 8 * sq.at, sq.phase, bound)) return false;
                if (i >= G::BUFS && !mbar_wait(dv_done + 8 * x, (i / G::BUFS - 1) & 1, bound)) return false;
                fence_after();
                mma_rows<DPAD>(tmem + x * BUF_COLS, base, ring(sq.at, 0), idesc_s, leader);
                mma_commit(s_full + 8 * x, leader);
                sq.next();
                return true;
            };
            const auto dprobs = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(full + 8 * (G::S0 + sg.at), sg.phase, bound)) return false;
                if (i >= G::BUFS && !mbar_wait(dk_done + 8 * x, (i / G::BUFS - 1) & 1, bound)) return false;
                fence_after();
                mma_rows<DPAD>(tmem + x * BUF_COLS + DP_COL, base + G::ROW_BYTES, ring(sg.at, 1), idesc_s, leader);
                mma_commit(dp_full + 8 * x, leader);
                sg.next();
                return true;
            };
            Turn<G::S1> vt;  // the tiles whose shares of dv and of dk are due
            Turn<G::S0> kt;
            const auto sums_v = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(p_full + 8 * x, (i / G::BUFS) & 1, bound)) return false;
                fence_after();
                mma_cols<DPAD>(tmem + DV_COL, tmem + x * BUF_COLS, 32, ring(vt.at, 1), idesc_o, i > 0, leader);
                mma_commit(dv_done + 8 * x, leader);
                mma_commit(empty + 8 * (G::S0 + vt.at), leader);
                vt.next();
                return true;
            };
            const auto sums_k = [&](int i) {
                const int x = i % G::BUFS;
                if (!mbar_wait(ds_full + 8 * x, (i / G::BUFS) & 1, bound)) return false;
                fence_after();
                mma_cols<DPAD>(tmem + DK_COL, tmem + x * BUF_COLS + DP_COL, 32, ring(kt.at, 0), idesc_o, i > 0, leader);
                mma_commit(dk_done + 8 * x, leader);
                mma_commit(empty + 8 * kt.at, leader);
                kt.next();
                return true;
            };
            bool ok = mbar_wait(row_full, 0, bound);
            for (int i = 0; i < G::BUFS && i < n; ++i) ok = ok && scores(i) && dprobs(i);
            if (G::BUFS == 1) {
                for (int i = 0; ok && i < n; ++i) {
                    const bool more = i + 1 < n;  // the next scores while dS is formed, the next dP behind dk
                    ok = sums_v(i) && (!more || scores(i + 1)) && sums_k(i) && (!more || dprobs(i + 1));
                }
            } else {
                // Each overwritten operand is awaited while the product after the one that reads it runs.
                for (int i = 0; ok && i < n; ++i) {
                    const bool more = i + 2 < n;
                    ok = sums_v(i) && sums_k(i) && (!more || (scores(i + 2) && dprobs(i + 2)));
                }
            }
            if (ok) mma_commit(acc_full, leader);  // else the elementwise warps' wait for it ends by the abort
            mma_commit(idle, leader);
            mbar_drain(idle, 0, f.timeout_ns);  // before the tensor memory is given back
        }
        __syncwarp();
    } else {
        // ---------------- elementwise: two threads a state, 32 queries each ----------------
        const int x = warp >> 3, half = (warp >> 2) & 1;  // x: the buffer of this group of warps
        const int64_t j = row0 + 32 * (warp & 3) + lane;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + x * BUF_COLS + 32 * half, tdp = ts + DP_COL;
        int64_t lo = 0, hi = 0;
        if (j < ny && nx > 0) column_cells(a, j, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        bool ok = true;
        Turn<G::S0> turn;
        int tile = x;
        if (x == 1) turn.next();
        for (int it = x; it < n; it += G::BUFS) {
            while (tile >= nq) tile -= nq;
            const uint32_t phase = (it / G::BUFS) & 1;
            if (!(ok = mbar_wait(full + 8 * turn.at, turn.phase, bound) && mbar_wait(s_full + 8 * x, phase, bound))) break;
            fence_after();
            const float* lse = stats + turn.at * 2 * kCols + 32 * half;
            const float* delta = lse + kCols;
            uint32_t s[32], p[32];
            tmem_ld32(ts, s);
            wait_ld();
            settle(s);
            const int off = (ia + tile) * kCols + 32 * half - ilo;
            const bool whole = __all_sync(kFull, off >= 0 && off + 32 <= width);
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                const float4 b4 = *reinterpret_cast<const float4*>(lse + c);
                s[c] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c]), a.scale_log2, b4.x)));
                s[c + 1] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 1]), a.scale_log2, b4.y)));
                s[c + 2] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 2]), a.scale_log2, b4.z)));
                s[c + 3] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[c + 3]), a.scale_log2, b4.w)));
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0;
            }
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]), T());
            tmem_st16(ts, w);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0 && !(f.stall == 3 && blockIdx.x == 0 && warp == 0 && it == 0)) mbar_arrive(p_full + 8 * x);
            if (!(ok = mbar_wait(dp_full + 8 * x, phase, bound))) break;
            fence_after();
            tmem_ld32(tdp, p);
            wait_ld();
            settle(p);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float4 d4 = *reinterpret_cast<const float4*>(delta + 2 * e);
                const float dd[4] = {d4.x, d4.y, d4.z, d4.w};
                float v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float dp = __uint_as_float(p[2 * e + y]);
                    v[y] = __uint_as_float(s[2 * e + y]) * (is_half<T> ? fmaf(dp, cf, -dd[y]) : dp - dd[y]);
                }
                w[e] = pack2(v[0], v[1], T());
                w[e + 1] = pack2(v[2], v[3], T());
            }
            tmem_st16(tdp, w);
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full + 8 * x);
            for (int y = 0; y < G::BUFS; ++y) turn.next();
            tile += G::BUFS;
        }
        if (ok && n > 0) ok = mbar_wait(acc_full, 0, bound);
        fence_after();
        // K's and V's places hold the rows on their way out: all products are done.
        const int64_t j0 = row0 + 32 * (warp & 3);
        const int64_t at = ((static_cast<int64_t>(b) * a.M + j0) * a.Hkv + hk) * a.d, pitch = static_cast<int64_t>(a.Hkv) * a.d;
        uint4* rows = reinterpret_cast<uint4*>(sm) + (warp & 3) * 32 * (DPAD / 8);
        const bool any = n > 0 && ok;
        if (x == 0)
            store_rows<T, DPAD>(tmem + lanes + DK_COL, rows, lane, half, 2 + (warp & 3), any, width > 0, !ok, a.scale * kPUnshift<T> / cf, f.dn,
                                a.d, static_cast<T*>(a.dk) + at, pitch, a.M - j0);
        if (x == G::BUFS - 1)
            store_rows<T, DPAD>(tmem + lanes + DV_COL, rows + G::ROW_BYTES / 16, lane, half, 6 + (warp & 3), any, width > 0, !ok,
                                kPUnshift<T>, f.dn, a.d, static_cast<T*>(a.dv) + at, pitch, a.M - j0);
        fence_before();
    }
    __syncthreads();
    if (warp == G::MMA_WARP) {
        fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
}

template <typename T, int DPAD>
cudaError_t backward_d(BwdArgs& f, cudaStream_t s)
{
    using G = Geom<DPAD>;
    const AttnArgs& a = f.a;
    constexpr bool half = is_half<T>;
    // As rows of a product (128 a tile) and as columns (64 a tile).
    CUtensorMap q_rows, g_rows, k_cols, v_cols, k_rows, v_rows, q_cols, g_cols;
    cudaError_t e = attention_bind_context();
    if (e != cudaSuccess) return e;
    if (!attention_tile_map(&q_rows, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, kTile) ||
        !attention_tile_map(&g_rows, half, a.dout, a.gs, a.B, a.N, a.Hq, a.d, kTile) ||
        !attention_tile_map(&k_cols, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, kCols) ||
        !attention_tile_map(&v_cols, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, kCols) ||
        !attention_tile_map(&k_rows, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, kTile) ||
        !attention_tile_map(&v_rows, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, kTile) ||
        !attention_tile_map(&q_cols, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, kCols) ||
        !attention_tile_map(&g_cols, half, a.dout, a.gs, a.B, a.N, a.Hq, a.d, kCols))
        return cudaErrorInvalidValue;
    static std::atomic<bool> allowed[3][128];
    const bool tail = DPAD == 64 && a.d <= 32;
    const auto dq = tail ? attend_dq_tc_kernel<T, DPAD, DPAD == 64> : attend_dq_tc_kernel<T, DPAD, false>;
    if ((e = allow_smem(dq, G::BYTES, allowed[tail ? 2 : 0])) != cudaSuccess) return e;
    if ((e = allow_smem(attend_dkdv_tc_kernel<T, DPAD>, G::BYTES, allowed[1])) != cudaSuccess) return e;
    f.tiles = static_cast<int>((a.N + kTile - 1) / kTile);
    dq<<<static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hq * f.tiles), G::THREADS, G::BYTES, s>>>(
        q_rows, g_rows, k_cols, v_cols, f);
    count_launch();
    f.tiles = static_cast<int>((a.M + kTile - 1) / kTile);
    attend_dkdv_tc_kernel<T, DPAD><<<static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hkv * f.tiles), G::THREADS, G::BYTES, s>>>(
        k_rows, v_rows, q_cols, g_cols, f);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t attention_tc_backward(const AttnArgs& a, bool bf16, cudaStream_t s)
{
    BwdArgs f{};
    f.a = a;
    f.timeout_ns = static_cast<uint64_t>(wait_timeout_s() * 1e9);
    f.dn = (a.d + 15) / 16 * 16;
    f.stall = attention_stall();
    if (bf16) return a.d <= 64 ? backward_d<__nv_bfloat16, 64>(f, s) : backward_d<__nv_bfloat16, 128>(f, s);
    return a.d <= 64 ? backward_d<__half, 64>(f, s) : backward_d<__half, 128>(f, s);
}

}  // namespace sdtw
