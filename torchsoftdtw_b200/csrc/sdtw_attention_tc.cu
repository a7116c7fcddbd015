// Cross attention of 16-bit operands on the tensor cores (tcgen05): forward.
//
// A CTA takes NT tiles of 128 query rows of one head and walks the 64-state tiles that their cells touch. Its
// warps specialise and meet only at mbarriers:
//   * eight softmax warps a row tile: two threads a row, 32 states each. S (128 x 64 fp32) is read from tensor memory,
//     masked where the tile leaves the row's interval, and P = 2^(s scale / ln 2 - m) goes back over it as 16-bit operand;
//   * one MMA warp a row tile: S = Q K^T (both from shared memory), O += P V (P from tensor memory, V read with its rows
//     as K). A row tile has two S buffers, so that the scores of the next state tile are there when a softmax ends;
//   * one TMA warp: Q once, then K and V tiles through a ring.
// The running maximum m is only raised, and O rescaled, when a row's scores outgrow it by 2^8: P stays below 2^8
// until then, and the final division by the row's sum makes it exact. (P is rounded to the operands' type for its product, which leaves
// out off by 1.1 to 1.5 times its own rounding; its sum is that of the 32-bit weights.) So a tile's weights are formed at once with the m of
// the tile before, beside its maximum, and formed again in the rare case that the maximum has outgrown it; the two threads
// of a row only have to agree on that, which one barrier with an OR does.
//
// Bound by the chain of a softmax step (wait, load of S, exponentials, meeting of a row's two threads, store of P), which two
// row tiles an SM, each with scores in hand, overlap in part: 2 x 4096 x 4096 x 16 x 128 bf16 270 us alone, 1020 TFLOP/s of 1718
// measured for a plain product, and 300 us (917) among others; 4 x 4096 x 4096 x 16 x 64 430 us, 640 TFLOP/s. Tiles of 64 states: S and O of two row tiles with
// two S buffers each fill tensor memory (d = 128). Exponentials as polynomials on the FMA pipe, an eighth to a half of them:
// no gain. Short series are bound by a CTA's start and end: 32 x 512 x 512 x 8 x 64 49 us, 350 TFLOP/s.
#include <mutex>
#include <type_traits>

#include "sdtw_attention.h"
#include "sdtw_attention_tc.h"
#include "sdtw_tc.cuh"

namespace sdtw {

using namespace tc;

namespace {

constexpr int kTile = 128;    // query rows a tile
constexpr int kStates = 64;   // states a tile
constexpr float kGrow = 8.f;  // log2 of what a row's scores may outgrow its m by

template <int DPAD, int NT>
struct Geom {
    static constexpr int Q_BYTES = kTile * DPAD * 2, KV_BYTES = kStates * DPAD * 2;
    static constexpr int Q_BLOCK = kTile * 128, KV_BLOCK = kStates * 128;  // 64 features of a tile
    static constexpr int NBLOCK = DPAD / 64;
    static constexpr int SLOTS = DPAD == 128 ? 9 : 8;
    static constexpr int OFF_RING = NT * Q_BYTES;
    static constexpr int OFF_ROW = OFF_RING + SLOTS * KV_BYTES;  // a number of each softmax thread's, for its partner
    static constexpr int OFF_BAR = OFF_ROW + NT * 256 * 4;
    // barriers: q_full, fix, ring full[SLOTS], ring empty[SLOTS], s_full[NT][2], p_full[NT][2], pv_full[NT],
    // o_full[NT], idle[NT]
    static constexpr int NBAR = 2 + 2 * SLOTS + 7 * NT;
    static constexpr int OFF_MISC = OFF_BAR + 8 * NBAR;  // tmem address, abort, tile ranges
    static constexpr int BYTES = OFF_MISC + 64 + 1024;   // and slack to align the base
    static constexpr uint32_t S_COL = 0;                 // S (and P over it): two buffers of 64 columns a row tile
    static constexpr uint32_t O_COL = NT * 2 * kStates;  // O: DPAD columns a row tile
    static constexpr uint32_t COLS_NEEDED = NT * (2 * kStates + DPAD);
    static constexpr uint32_t TMEM_COLS = COLS_NEEDED <= 256 ? 256 : 512;
    static constexpr int SOFTMAX_WARPS = 8 * NT;
    static constexpr int TMA_WARP = SOFTMAX_WARPS + NT;
    static constexpr int THREADS = 32 * (TMA_WARP + 1);
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

struct FwdArgs {
    AttnArgs a;
    uint64_t timeout_ns;
    int tiles;     // CTAs a head: ceil(N / (128 NT))
    int dn;        // d rounded up to 16: columns of O
    int negative;  // scale < 0: the scores change sign
    int stall;     // attention_stall() == 1
};

template <typename T, int DPAD, int NT>
__global__ void __launch_bounds__(Geom<DPAD, NT>::THREADS, NT == 1 ? 2 : 1)
    attend_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ FwdArgs f)
{
    using G = Geom<DPAD, NT>;
    const AttnArgs& a = f.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(sm);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t q_full = base + G::OFF_BAR, fix = q_full + 8, full = fix + 8, empty = full + 8 * G::SLOTS;
    const uint32_t s_full = empty + 8 * G::SLOTS, p_full = s_full + 16 * NT, pv_full = p_full + 16 * NT, o_full = pv_full + 8 * NT, idle = o_full + 8 * NT;
    uint32_t* misc = reinterpret_cast<uint32_t*>(sm + G::OFF_MISC);
    volatile int* ranges = reinterpret_cast<volatile int*>(misc + 2);  // first and last + 1 state tile of each tile
    const Bound bound{f.timeout_ns, reinterpret_cast<volatile int*>(misc + 1), a.err};

    const int64_t id = blockIdx.x;
    const int qt = static_cast<int>(id % f.tiles);
    const int h = static_cast<int>(id / f.tiles % a.Hq), b = static_cast<int>(id / f.tiles / a.Hq);
    const int hk = h / a.group;
    const int row0 = qt * kTile * NT;
    int64_t nx, ny;
    const bool good = pair_lengths(a, b, nx, ny);

    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(fix, 1);
        for (int s = 0; s < G::SLOTS; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, NT);  // every MMA warp passes every tile
        }
        for (int w = 0; w < NT; ++w) {
            for (int x = 0; x < 2; ++x) {
                mbar_init(s_full + 16 * w + 8 * x, 1);
                mbar_init(p_full + 16 * w + 8 * x, 8);
            }
            mbar_init(pv_full + 8 * w, 1);
            mbar_init(o_full + 8 * w, 1);
            mbar_init(idle + 8 * w, 1);
            const int64_t r0 = row0 + w * kTile;
            int first = 0, last = 0;
            if (r0 < nx && ny > 0) {
                const int64_t r1 = r0 + kTile < nx ? r0 + kTile : nx;
                int64_t lo, hi, lo1, hi1;
                row_cells(a, r0, nx, ny, lo, hi);
                row_cells(a, r1 - 1, nx, ny, lo1, hi1);
                first = static_cast<int>(lo / kStates);
                last = static_cast<int>((hi1 + kStates - 1) / kStates);
            }
            ranges[2 * w] = first;
            ranges[2 * w + 1] = last;
        }
        *bound.abort = 0;
        if (!good) atomicOr(a.err, kErrBadLength);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == G::SOFTMAX_WARPS) tmem_alloc(base + G::OFF_MISC, G::TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
    int first[NT], last[NT], ja = 1 << 30, jb = 0;
#pragma unroll
    for (int w = 0; w < NT; ++w) {
        first[w] = ranges[2 * w];
        last[w] = ranges[2 * w + 1];
        if (last[w] > first[w]) {
            ja = min(ja, first[w]);
            jb = max(jb, last[w]);
        }
    }

    const int count = jb > ja ? jb - ja : 0;  // state tiles
    if (warp == G::TMA_WARP) {
        // ---------------- TMA ----------------
        if (count > 0) {
            if (lane == 0) {
                uint32_t bytes = 0;
                for (int w = 0; w < NT; ++w)
                    if (last[w] > first[w]) bytes += G::Q_BYTES;
                mbar_expect_tx(q_full, bytes);
                for (int w = 0; w < NT; ++w)
                    if (last[w] > first[w])
                        for (int x = 0; x < G::NBLOCK; ++x)
                            tma_load_4d(base + w * G::Q_BYTES + x * G::Q_BLOCK, &mq, q_full, 64 * x, row0 + w * kTile, h, b);
            }
            int issued = 0;
            const auto load = [&](int j, bool is_v) {
                const int n = issued, slot = n % G::SLOTS;
                if (n >= G::SLOTS && !mbar_wait(empty + 8 * slot, (n / G::SLOTS - 1) & 1, bound)) return false;
                const int at = G::OFF_RING + slot * G::KV_BYTES;
                // V rows past the length meet weights of zero, but may hold NaN: the tile that the length ends in
                // is cleared behind it before it is handed on (once a CTA: the last one).
                const int64_t left = ny - static_cast<int64_t>(j) * kStates;
                const bool clear = is_v && left < kStates && ny < a.M;
                const uint32_t bar = clear ? fix : full + 8 * slot;
                if (lane == 0) {
                    mbar_expect_tx(bar, G::KV_BYTES);
                    for (int x = 0; x < G::NBLOCK; ++x)
                        tma_load_4d(base + at + x * G::KV_BLOCK, is_v ? &mv : &mk, bar, 64 * x, j * kStates, hk, b);
                }
                __syncwarp();
                bool ok = true;
                if (clear) {
                    ok = mbar_wait(fix, 0, bound);
                    if (!ok) mbar_drain(fix, 0, f.timeout_ns);  // `full`, drained below, will not tell of this load
                    for (int x = 0; x < G::NBLOCK; ++x)
                        for (int u = static_cast<int>(left) * 8 + lane; u < kStates * 8; u += 32)
                            *reinterpret_cast<uint4*>(sm + at + x * G::KV_BLOCK + 16 * u) = make_uint4(0, 0, 0, 0);
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * slot);
                }
                issued = n + 1;
                return ok;
            };
            // In the order of use: K 0, K 1, then V t and K t + 2.
            bool ok = load(ja, false) && (count < 2 || load(ja + 1, false));
            for (int t = 0; t < count && ok; ++t) ok = load(ja + t, true) && (t + 2 >= count || load(ja + t + 2, false));
            // Every load has landed before the CTA ends (also after an abort).
            mbar_drain(q_full, 0, f.timeout_ns);
            for (int n = issued < G::SLOTS ? 0 : issued - G::SLOTS; n < issued; ++n)
                mbar_drain(full + 8 * (n % G::SLOTS), (n / G::SLOTS) & 1, f.timeout_ns);
        }
    } else if (warp >= G::SOFTMAX_WARPS) {
        // ---------------- MMA, one warp a row tile ----------------
        const int w = warp - G::SOFTMAX_WARPS;
        if (count > 0) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(kStates, false);
            const uint32_t idesc_o = mma_idesc<T>(f.dn, true);
            const int ja_w = NT == 1 || w == 0 ? first[0] : first[NT - 1];
            const int jb_w = NT == 1 || w == 0 ? last[0] : last[NT - 1];
            const uint64_t qd = desc_k(base + w * G::Q_BYTES);
            const uint32_t s_col = tmem + G::S_COL + 2 * w * kStates, o_col = tmem + G::O_COL + w * DPAD;
            int slot = 0;
            uint32_t phase = 0;
            bool ok = mbar_wait(q_full, 0, bound);
            const auto arrived = [&] { return mbar_wait(full + 8 * slot, phase, bound); };
            const auto release = [&] {  // behind the products that read the slot
                mma_commit(empty + 8 * slot, leader);
                if (++slot == G::SLOTS) {
                    slot = 0;
                    phase ^= 1;
                }
            };
            // The scores of state tile j into the buffer of its turn. Products complete in no promised order among
            // themselves, so the PV product that read the weights there has to be awaited.
            const auto scores = [&](int j) {
                const int it = j - ja_w, x = it & 1;
                if (it >= 2) ok = mbar_wait(pv_full + 8 * w, it & 1, bound) && ok;
                ok = ok && arrived();
                if (!ok) return;
                fence_after();
                const uint64_t kd = desc_k(base + G::OFF_RING + slot * G::KV_BYTES);
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k)  // features past d are zero; a branch between products costs more
                    mma_ss(s_col + x * kStates, desc_at(qd, (k / 4) * G::Q_BLOCK + (k % 4) * 32),
                           desc_at(kd, (k / 4) * G::KV_BLOCK + (k % 4) * 32), idesc_s, k > 0, leader);
                mma_commit(s_full + 16 * w + 8 * x, leader);
            };
            // In the order of the loads: K 0, K 1, then V t and K t + 2. A tile outside this row tile's range (it only
            // bridges the CTA's two) is passed on when it has landed.
            for (int t = 0; ok && t < 2 && t < count; ++t) {
                if (ja + t >= ja_w && ja + t < jb_w)
                    scores(ja + t);
                else
                    ok = arrived();
                release();
            }
            for (int t = 0; ok && t < count; ++t) {
                const int j = ja + t;
                ok = arrived();
                if (ok && j >= ja_w && j < jb_w) {
                    const int it = j - ja_w, x = it & 1;
                    if (!(ok = mbar_wait(p_full + 16 * w + 8 * x, (it >> 1) & 1, bound))) break;
                    fence_after();
                    const uint64_t vd = desc_mn(base + G::OFF_RING + slot * G::KV_BYTES, G::KV_BLOCK);
#pragma unroll
                    for (int k = 0; k < kStates / 16; ++k)
                        mma_ts(o_col, s_col + x * kStates + 8 * k, desc_at(vd, 2048 * k), idesc_o, k > 0 || it > 0, leader);
                    mma_commit(pv_full + 8 * w, leader);
                    if (j + 1 == jb_w) mma_commit(o_full + 8 * w, leader);
                }
                release();
                if (ok && t + 2 < count) {
                    if (j + 2 >= ja_w && j + 2 < jb_w)
                        scores(j + 2);
                    else
                        ok = arrived();
                    release();
                }
            }
            // All products have completed before the tensor memory is given back.
            mma_commit(idle + 8 * w, leader);
            mbar_drain(idle + 8 * w, 0, f.timeout_ns);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: two threads a row, 32 states of a tile each ----------------
        const int w = NT == 1 ? 0 : warp >> 3, half = (warp >> 2) & 1;
        const int row = 32 * (warp & 3) + lane, pair = 1 + 4 * w + (warp & 3);  // the pair's named barrier
        const int64_t i = row0 + w * kTile + row;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts0 = tmem + lanes + G::S_COL + 2 * w * kStates, to = tmem + lanes + G::O_COL + w * DPAD;
        float* mine = reinterpret_cast<float*>(sm + G::OFF_ROW) + w * 256 + half * 128 + row;
        const float* theirs = reinterpret_cast<float*>(sm + G::OFF_ROW) + w * 256 + (1 - half) * 128 + row;
        const auto meet = [&] { asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair) : "memory"); };
        const auto either = [&](bool x) {
            uint32_t r;
            asm volatile(
                "{ .reg .pred p, q; setp.ne.b32 p, %1, 0; barrier.cta.red.or.pred q, %2, 64, p; selp.b32 %0, 1, 0, q; }"
                : "=r"(r)
                : "r"(static_cast<uint32_t>(x)), "r"(pair)
                : "memory");
            return r != 0;
        };
        int64_t lo = 0, hi = 0;
        if (i < nx && ny > 0) row_cells(a, i, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        const int ja_w = NT == 1 ? first[0] : (w ? first[NT - 1] : first[0]);
        const int jb_w = NT == 1 ? last[0] : (w ? last[NT - 1] : last[0]);
        const float sl = a.scale_log2;
        // fp16 weights are kept 2^6 larger, so that weights down to 2^-20 of a row's largest stay normal numbers.
        constexpr float kShift = std::is_same<T, __half>::value ? 6.f : 0.f;
        float m = -INFINITY, bias = 0.f, sum = 0.f;
        bool ok = true;  // the same in both threads of a row from each meeting on
        for (int j = ja_w; j < jb_w; ++j) {
            const int it = j - ja_w;
            const uint32_t ts = ts0 + (it & 1) * kStates;
            ok = ok && mbar_wait(s_full + 16 * w + 8 * (it & 1), (it >> 1) & 1, bound);
            fence_after();
            const int off = j * kStates + 32 * half - ilo;
            const bool whole = __all_sync(kFull, off >= 0 && off + 32 <= width);
            uint32_t s[32], p[16];
            tmem_ld32(ts + 32 * half, s);
            wait_ld();
            settle(s);
            if (f.negative) {
#pragma unroll
                for (int c = 0; c < 32; ++c) s[c] ^= 0x80000000u;
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0xff800000u;
            }
            float t0 = m, t1 = __uint_as_float(s[0]), t2 = __uint_as_float(s[1]), t3 = __uint_as_float(s[2]);
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                t0 = fmaxf(t0, __uint_as_float(s[c]));
                t1 = fmaxf(t1, __uint_as_float(s[c + 1]));
                t2 = fmaxf(t2, __uint_as_float(s[c + 2]));
                t3 = fmaxf(t3, __uint_as_float(s[c + 3]));
            }
            float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
            float tile = 0.f;
            const auto weights = [&] {  // P and its sum with the present m
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = ex2f(fmaf(__uint_as_float(s[2 * e]), sl, bias));
                    const float y = ex2f(fmaf(__uint_as_float(s[2 * e + 1]), sl, bias));
                    l0 += x;
                    l1 += y;
                    p[e] = pack2(x, y, T());
                }
                tile = l0 + l1;
            };
            if (it > 0) weights();
            // Both warps have read their scores when they meet here: P may overwrite them.
            if (either(it == 0 || !ok || (top - m) * sl > kGrow)) {
                *mine = ok ? top : __int_as_float(0x7fc00000);
                meet();
                const float other = *theirs;
                meet();
                if (!ok || __any_sync(kFull, other != other)) {  // this warp gave up, or its partner did (a maximum is no NaN)
                    ok = false;
                    break;
                }
                top = fmaxf(top, other);
                if (it > 0) {
                    // O holds the sum of the tiles before, once their products have completed. Its features go by 16 to
                    // the two threads of the row.
                    ok = mbar_wait(pv_full + 8 * w, (it - 1) & 1, bound);
                    fence_after();
                    const float fix_up = top == -INFINITY ? 1.f : ex2f((m - top) * sl);
                    sum *= fix_up;
                    for (int c = 16 * half; c < f.dn; c += 32) {
                        uint32_t o[16];
                        tmem_ld16(to + c, o);
                        wait_ld();
                        settle(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix_up);
                        tmem_st16(to + c, o);
                    }
                }
                m = top;
                bias = m == -INFINITY ? 0.f : fmaf(-m, sl, kShift);
                weights();
            }
            tmem_st16(ts + 16 * half, p);
            sum += tile;
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0 && !(f.stall && blockIdx.x == 0 && warp == 0 && it == 0)) mbar_arrive(p_full + 16 * w + 8 * (it & 1));
        }
        // (Not pv_full: PV products of this tile and the one before may both have completed by now, or neither, and a
        // parity tells a phase only from its neighbours.)
        if (ok && jb_w > ja_w) ok = mbar_wait(o_full + 8 * w, 0, bound);
        fence_after();
        *mine = sum;
        ok = !either(!ok);
        sum += *theirs;
        // Rows without a cell are zero; a bad sample's, and all after a wait that ran out, NaN. A pair of warps lays its 32
        // rows down in shared memory (Q's place; all scores are done) in 16-byte units, turned by the row against bank
        // conflicts, and stores them row by row.
        const float scale = width > 0 ? 1.f / sum : 0.f;
        const bool any = jb_w > ja_w && ok;
        const bool broken = !ok || !good;
        constexpr int UPR = DPAD / 8;  // units a row
        uint4* rows = reinterpret_cast<uint4*>(sm + w * G::Q_BYTES) + (warp & 3) * 32 * UPR;
        const int64_t i0 = row0 + w * kTile + 32 * (warp & 3);
        for (int part = 0; part < (a.out_lo ? 2 : 1); ++part) {
            for (int c = 16 * half; c < f.dn; c += 32) {
                uint32_t o[16];
                if (any) {
                    tmem_ld16(to + c, o);
                    wait_ld();
                    settle(o);
                }
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    uint32_t v[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float v0 = any && width > 0 ? __uint_as_float(o[e + 2 * x]) * scale : 0.f;
                        float v1 = any && width > 0 ? __uint_as_float(o[e + 2 * x + 1]) * scale : 0.f;
                        if (broken) v0 = v1 = __int_as_float(0x7fc00000);
                        v[x] = pack2(v0, v1, T());
                        if (part == 1) {
                            const T* r = reinterpret_cast<const T*>(&v[x]);
                            v[x] = pack2((v0 - to_f(r[0])) * kLoScale<T>, (v1 - to_f(r[1])) * kLoScale<T>, T());
                        }
                    }
                    rows[lane * UPR + (((c + e) / 8) ^ (lane & 7))] = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
            meet();
            T* out = static_cast<T*>(part ? a.out_lo : a.out) + ((static_cast<int64_t>(b) * a.N + i0) * a.Hq + h) * a.d;
            const int64_t pitch = static_cast<int64_t>(a.Hq) * a.d;
#pragma unroll 4
            for (int r = half * (32 / UPR) + lane / UPR; r < 32; r += 2 * (32 / UPR))
                if (i0 + r < a.N && lane % UPR * 8 < a.d)
                    *reinterpret_cast<uint4*>(out + r * pitch + lane % UPR * 8) = rows[r * UPR + ((lane % UPR) ^ (r & 7))];
            meet();
        }
        if (half == 0 && i < a.N && a.lse)
            a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.N + i] = width > 0 ? fmaf(m, sl, log2f(sum) - kShift) : -INFINITY;
        fence_before();
    }
    __syncthreads();
    if (warp == G::SOFTMAX_WARPS) {
        fence_after();
        tmem_free(tmem, G::TMEM_COLS);
    }
}

// ---- host ----
std::mutex g_mu;
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

cudaError_t get_encode(PFN_cuTensorMapEncodeTiled_v12000& fn)
{
    std::lock_guard<std::mutex> lock(g_mu);
    if (!g_encode) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
        if (e != cudaSuccess) return e;
        if (q != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
        g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    fn = g_encode;
    return cudaSuccess;
}

template <typename T, int DPAD, int NT>
cudaError_t launch_forward(FwdArgs& f, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s)
{
    using G = Geom<DPAD, NT>;
    static std::atomic<bool> allowed[128];
    const cudaError_t e = allow_smem(attend_tc_kernel<T, DPAD, NT>, G::BYTES, allowed);
    if (e != cudaSuccess) return e;
    f.tiles = static_cast<int>((f.a.N + kTile * NT - 1) / (kTile * NT));
    const int64_t grid = static_cast<int64_t>(f.a.B) * f.a.Hq * f.tiles;
    attend_tc_kernel<T, DPAD, NT><<<static_cast<unsigned>(grid), G::THREADS, G::BYTES, s>>>(mq, mk, mv, f);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward_t(const AttnArgs& a, cudaStream_t s)
{
    const cudaError_t bound = attention_bind_context();
    if (bound != cudaSuccess) return bound;
    CUtensorMap mq, mk, mv;
    constexpr bool half = std::is_same<T, __half>::value;
    if (!attention_tile_map(&mq, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, kTile) ||
        !attention_tile_map(&mk, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, kStates) ||
        !attention_tile_map(&mv, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, kStates))
        return cudaErrorInvalidValue;
    FwdArgs f{};
    f.a = a;
    f.timeout_ns = static_cast<uint64_t>(wait_timeout_s() * 1e9);
    f.dn = (a.d + 15) / 16 * 16;
    f.negative = a.scale_log2 < 0;
    f.stall = attention_stall() == 1;
    f.a.scale_log2 = fmaxf(fabsf(a.scale_log2), 1e-30f);  // a scale of zero: all scores equal
    if (a.d <= 64) return launch_forward<T, 64, 1>(f, mq, mk, mv, s);
    return launch_forward<T, 128, 2>(f, mq, mk, mv, s);
}

}  // namespace

namespace {
std::atomic<int> g_stall{0};
}
int attention_stall() { return g_stall.load(std::memory_order_relaxed); }

cudaError_t attention_bind_context()
{
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e == cudaSuccess ? cudaSetDevice(dev) : e;
}

bool attention_tile_map(CUtensorMap* map, bool half, const void* ptr, const Strides& st, int64_t B, int64_t rows, int64_t H,
                        int64_t d, int box_rows)
{
    PFN_cuTensorMapEncodeTiled_v12000 encode;
    if (get_encode(encode) != cudaSuccess) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(H),
                                static_cast<cuuint64_t>(B)};
    // The stride of a dimension of size one is never used, and may be anything in the caller's tensor.
    const auto bytes = [](int64_t s, int64_t size) { return static_cast<cuuint64_t>(size == 1 ? 16 : s * 2); };
    const cuuint64_t strides[3] = {bytes(st.n, rows), bytes(st.h, H), bytes(st.b, B)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr),
                  dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool attention_tc_takes(const void* p, const Strides& st, int64_t B, int64_t rows, int64_t H, int64_t d)
{
    const auto fits = [](int64_t s, int64_t size) { return size == 1 || (s > 0 && s % 8 == 0 && s < (int64_t{1} << 38)); };
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && d % 8 == 0 && fits(st.n, rows) && fits(st.h, H) && fits(st.b, B);
}

cudaError_t attention_tc_forward(const AttnArgs& a, bool bf16, cudaStream_t s)
{
    return bf16 ? forward_t<__nv_bfloat16>(a, s) : forward_t<__half>(a, s);
}

}  // namespace sdtw

// Test hook (see attention_stall).
extern "C" void sdtw_debug_attention_stall(int which) { sdtw::g_stall.store(which); }
