// Cross attention of 16-bit operands on the tensor cores (tcgen05): forward.
//
// A CTA takes NT tiles of 128 query rows of one head and walks the 128-state tiles that their cells touch. Its
// warps specialise and meet only at mbarriers:
//   * four softmax warps a tile: one row a thread. S (128 x 128 fp32) is read from tensor memory, masked where
//     the tile leaves the row's interval, and P = 2^(s scale / ln 2 - m) goes back over it as 16-bit operand;
//   * one MMA warp: S = Q K^T (both from shared memory), O += P V (P from tensor memory, V read with its rows as
//     K), issued so that one tile's products run while the other tile's softmax does;
//   * one TMA warp: Q once, then K and V tiles through a ring.
// The running maximum m is only raised, and O rescaled, when a row's scores outgrow it by 2^8: P stays below 2^8
// until then, and the final division by the row's sum makes it exact. With two tiles (NT = 2) every K and V tile
// is read once for 256 rows and the two tiles' products and softmaxes alternate on their units.
#include <mutex>
#include <type_traits>

#include "sdtw_attention.h"
#include "sdtw_attention_tc.h"
#include "sdtw_tc.cuh"

namespace sdtw {

using namespace tc;

namespace {

constexpr int kTile = 128;  // query rows and states a tile
constexpr float kGrow = 8.f;  // log2 of what a row's scores may outgrow its m by

template <int DPAD, int NT>
struct Geom {
    static constexpr int TILE_BYTES = kTile * DPAD * 2;
    static constexpr int BLOCK = kTile * 128;  // 64 features of a tile
    static constexpr int NBLOCK = DPAD / 64;
    static constexpr int SLOTS = NT == 2 ? (DPAD == 128 ? 5 : 8) : 4;
    static constexpr int OFF_RING = NT * TILE_BYTES;
    static constexpr int OFF_BAR = OFF_RING + SLOTS * TILE_BYTES;
    // barriers: q_full, fix, ring full[SLOTS], ring empty[SLOTS], s_full[NT], p_full[NT], o_full[NT]
    static constexpr int NBAR = 2 + 2 * SLOTS + 3 * NT;
    static constexpr int OFF_MISC = OFF_BAR + 8 * NBAR;  // tmem address, abort, tile ranges
    static constexpr int BYTES = OFF_MISC + 64 + 1024;   // and slack to align the base
    static constexpr uint32_t S_COL = 0;                 // S (and P over it): 128 columns a tile
    static constexpr uint32_t O_COL = NT * kTile;        // O: DPAD columns a tile
    static constexpr uint32_t COLS_NEEDED = NT * (kTile + DPAD);
    static constexpr uint32_t TMEM_COLS = COLS_NEEDED <= 256 ? 256 : 512;
    static constexpr int SOFTMAX_WARPS = 4 * NT;
    static constexpr int THREADS = 32 * (SOFTMAX_WARPS + 2);
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

struct FwdArgs {
    AttnArgs a;
    uint64_t timeout_ns;
    int tiles;     // CTAs a head: ceil(N / (128 NT))
    int dn;        // d rounded up to 16: columns of O
    int negative;  // scale < 0: the scores change sign
};

// 16-bit results of one row, from `v` times `f`: features c .. c + 31 that lie below d. The residual row (may be
// null) takes what the rounding dropped.
template <typename T>
__device__ __forceinline__ void store_row32(T* row, T* lo, const float (&v)[32], int c, int d)
{
    if (d % 8 == 0) {  // rows start on 16 bytes
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            if (c + i >= d) break;
            uint32_t w[4], r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = v[i + 2 * e], y = v[i + 2 * e + 1];
                w[e] = pack2(x, y, T());
                const T* h = reinterpret_cast<const T*>(&w[e]);
                r[e] = pack2(x - to_f(h[0]), y - to_f(h[1]), T());
            }
            *reinterpret_cast<uint4*>(row + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
            if (lo) *reinterpret_cast<uint4*>(lo + c + i) = make_uint4(r[0], r[1], r[2], r[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (c + i < d) {
                const T h = from_f<T>(v[i]);
                row[c + i] = h;
                if (lo) lo[c + i] = from_f<T>(v[i] - to_f(h));
            }
    }
}

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
    const uint32_t s_full = empty + 8 * G::SLOTS, p_full = s_full + 8 * NT, o_full = p_full + 8 * NT;
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
            mbar_init(empty + 8 * s, 1);
        }
        for (int w = 0; w < NT; ++w) {
            mbar_init(s_full + 8 * w, 1);
            mbar_init(p_full + 8 * w, 4);
            mbar_init(o_full + 8 * w, 1);
            const int64_t r0 = row0 + w * kTile;
            int first = 0, last = 0;
            if (r0 < nx && ny > 0) {
                const int64_t r1 = r0 + kTile < nx ? r0 + kTile : nx;
                int64_t lo, hi, lo1, hi1;
                row_cells(a, r0, nx, ny, lo, hi);
                row_cells(a, r1 - 1, nx, ny, lo1, hi1);
                first = static_cast<int>(lo / kTile);
                last = static_cast<int>((hi1 + kTile - 1) / kTile);
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

    if (warp == G::SOFTMAX_WARPS + 1) {
        // ---------------- TMA ----------------
        int issued = 0;
        bool ok = true;
        if (ja < jb) {
            if (lane == 0) {
                uint32_t bytes = 0;
                for (int w = 0; w < NT; ++w)
                    if (last[w] > first[w]) bytes += G::TILE_BYTES;
                mbar_expect_tx(q_full, bytes);
                for (int w = 0; w < NT; ++w)
                    if (last[w] > first[w])
                        for (int x = 0; x < G::NBLOCK; ++x)
                            tma_load_4d(base + w * G::TILE_BYTES + x * G::BLOCK, &mq, q_full, 64 * x, row0 + w * kTile, h, b);
            }
            for (int n = 0; n < 2 * (jb - ja) && ok; ++n) {  // K and V of each state tile
                const int j = ja + n / 2, slot = n % G::SLOTS;
                const bool is_v = n & 1;
                if (n >= G::SLOTS && !mbar_wait(empty + 8 * slot, (n / G::SLOTS - 1) & 1, bound)) {
                    ok = false;
                    break;
                }
                const uint32_t dst = base + G::OFF_RING + slot * G::TILE_BYTES;
                // V rows past the length meet weights of zero, but may hold NaN: the tile that the length ends in
                // is cleared behind it before it is handed on.
                const int64_t left = ny - static_cast<int64_t>(j) * kTile;
                const bool clear = is_v && left < kTile && ny < a.M;
                const uint32_t bar = clear ? fix : full + 8 * slot;
                if (lane == 0) {
                    mbar_expect_tx(bar, G::TILE_BYTES);
                    for (int x = 0; x < G::NBLOCK; ++x)
                        tma_load_4d(dst + x * G::BLOCK, is_v ? &mv : &mk, bar, 64 * x, j * kTile, hk, b);
                }
                __syncwarp();
                if (clear) {  // once a CTA: only the last state tile can end inside
                    if (!mbar_wait(fix, 0, bound)) ok = false;
                    const int skip = static_cast<int>(left) * 8;  // 16-byte units a 64-feature block
                    unsigned char* at = sm + G::OFF_RING + slot * G::TILE_BYTES;
                    for (int x = 0; x < G::NBLOCK; ++x)
                        for (int u = skip + lane; u < kTile * 8; u += 32)
                            *reinterpret_cast<uint4*>(at + x * G::BLOCK + 16 * u) = make_uint4(0, 0, 0, 0);
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * slot);
                }
                issued = n + 1;
            }
            // Every load has landed before the CTA ends (also after an abort).
            mbar_drain(q_full, 0, f.timeout_ns);
            for (int n = issued < G::SLOTS ? 0 : issued - G::SLOTS; n < issued; ++n)
                mbar_drain(full + 8 * (n % G::SLOTS), (n / G::SLOTS) & 1, f.timeout_ns);
        }
    } else if (warp == G::SOFTMAX_WARPS) {
        // ---------------- MMA ----------------
        if (ja < jb) {
            const uint32_t leader = elect_leader();
            const uint32_t idesc_s = mma_idesc<T>(kTile, false);
            const uint32_t idesc_o = mma_idesc<T>(f.dn, true);
            const int ksteps = f.dn / 16;
            uint32_t used[NT] = {};  // P tiles consumed
            bool ok = mbar_wait(q_full, 0, bound);
            const auto ring = [&](int n) { return mbar_wait(full + 8 * (n % G::SLOTS), (n / G::SLOTS) & 1, bound); };
            const auto slot_at = [&](int n) { return base + G::OFF_RING + (n % G::SLOTS) * G::TILE_BYTES; };
            const auto scores = [&](int w, int n) {
                const uint64_t qd = desc_k(base + w * G::TILE_BYTES), kd = desc_k(slot_at(n));
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k) {
                    const uint32_t at = (k / 4) * G::BLOCK + (k % 4) * 32;
                    if (k < ksteps)
                        mma_ss(tmem + G::S_COL + w * kTile, desc_at(qd, at), desc_at(kd, at), idesc_s, k > 0, leader);
                }
                mma_commit(s_full + 8 * w, leader);
            };
            if (ok && (ok = ring(0))) {
                fence_after();
#pragma unroll
                for (int w = 0; w < NT; ++w)
                    if (ja >= first[w] && ja < last[w]) scores(w, 0);
                mma_commit(empty, leader);
            }
            for (int j = ja; ok && j < jb; ++j) {
                const int nv = 2 * (j - ja) + 1, nk = nv + 1;
                bool have_v = false, have_k = false;
#pragma unroll
                for (int w = 0; w < NT; ++w) {
                    if (!ok) break;
                    if (j >= first[w] && j < last[w]) {
                        if (!have_v) have_v = ok = ring(nv);
                        if (ok) ok = mbar_wait(p_full + 8 * w, used[w] & 1, bound);
                        if (!ok) break;
                        fence_after();
                        const uint64_t vd = desc_mn(slot_at(nv), G::BLOCK);
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            mma_ts(tmem + G::O_COL + w * DPAD, tmem + G::S_COL + w * kTile + 8 * k, desc_at(vd, 2048 * k),
                                   idesc_o, k > 0 || used[w] > 0, leader);
                        ++used[w];
                        if (j + 1 >= last[w]) mma_commit(o_full + 8 * w, leader);
                    }
                    if (j + 1 >= first[w] && j + 1 < last[w]) {
                        if (!have_k) have_k = ok = ring(nk);
                        if (!ok) break;
                        fence_after();
                        scores(w, nk);
                    }
                }
                if (!ok) break;
                // The commits also cover slots that no tile read (they only bridge two tiles' ranges).
                if (!have_v && !(ok = ring(nv))) break;
                mma_commit(empty + 8 * (nv % G::SLOTS), leader);
                if (j + 1 < jb) {
                    if (!have_k && !(ok = ring(nk))) break;
                    mma_commit(empty + 8 * (nk % G::SLOTS), leader);
                }
            }
            // All products have completed before the tensor memory is given back.
            mma_commit(fix, leader);
            mbar_drain(fix, (ny < a.M && jb > ja && ny - static_cast<int64_t>(jb - 1) * kTile < kTile) ? 1 : 0, f.timeout_ns);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: one row a thread ----------------
        const int w = NT == 1 ? 0 : warp >> 2;
        const int64_t i = row0 + w * kTile + (tid & 127);
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + G::S_COL + w * kTile, to = tmem + lanes + G::O_COL + w * DPAD;
        int64_t lo = 0, hi = 0;
        if (i < nx && ny > 0) row_cells(a, i, nx, ny, lo, hi);
        const int ilo = static_cast<int>(lo), width = static_cast<int>(hi - lo);
        const int ja_w = NT == 1 ? first[0] : (w ? first[NT - 1] : first[0]);
        const int jb_w = NT == 1 ? last[0] : (w ? last[NT - 1] : last[0]);
        const float sl = a.scale_log2;
        // fp16 weights are kept 2^6 larger, so that weights down to 2^-20 of a row's largest stay normal numbers.
        constexpr float kShift = std::is_same<T, __half>::value ? 6.f : 0.f;
        float m = -INFINITY, sum = 0.f;
        bool ok = true;
        for (int j = ja_w; j < jb_w; ++j) {
            const int it = j - ja_w;
            if (!mbar_wait(s_full + 8 * w, it & 1, bound)) {
                ok = false;
                break;
            }
            fence_after();
            uint32_t s[kTile];
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tmem_ld32(ts + c, s + c);
            wait_ld();
            settle(s);
            if (f.negative) {
#pragma unroll
                for (int c = 0; c < kTile; ++c) s[c] ^= 0x80000000u;
            }
            const int off = j * kTile - ilo;
            if (!__all_sync(kFull, off >= 0 && off + kTile <= width)) {
#pragma unroll
                for (int c = 0; c < kTile; ++c)
                    if (static_cast<unsigned>(off + c) >= static_cast<unsigned>(width)) s[c] = 0xff800000u;
            }
            float t0 = __uint_as_float(s[0]), t1 = __uint_as_float(s[1]);
            float t2 = __uint_as_float(s[2]), t3 = __uint_as_float(s[3]);
#pragma unroll
            for (int c = 4; c < kTile; c += 4) {
                t0 = fmaxf(t0, __uint_as_float(s[c]));
                t1 = fmaxf(t1, __uint_as_float(s[c + 1]));
                t2 = fmaxf(t2, __uint_as_float(s[c + 2]));
                t3 = fmaxf(t3, __uint_as_float(s[c + 3]));
            }
            const float m2 = fmaxf(m, fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)));
            if (it == 0) {
                m = m2;
            } else if (__any_sync(kFull, (m2 - m) * sl > kGrow)) {
                // O holds the sum of the tiles before (their products completed before this tile's scores).
                const float fix_up = m2 == -INFINITY ? 1.f : ex2f((m - m2) * sl);
                m = m2;
                sum *= fix_up;
                for (int c = 0; c < f.dn; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(to + c, o);
                    wait_ld();
                    settle(o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix_up);
                    tmem_st16(to + c, o);
                }
            }
            const float bias = m == -INFINITY ? 0.f : fmaf(-m, sl, kShift);
            float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = ex2f(fmaf(__uint_as_float(s[c + 2 * e]), sl, bias));
                    const float y = ex2f(fmaf(__uint_as_float(s[c + 2 * e + 1]), sl, bias));
                    l0 += x;
                    l1 += y;
                    p[e] = pack2(x, y, T());
                }
                tmem_st16(ts + c / 2, p);
            }
            sum += l0 + l1;
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * w);
        }
        if (ok && jb_w > ja_w) ok = mbar_wait(o_full + 8 * w, 0, bound);
        fence_after();
        ok = __all_sync(kFull, ok);
        // Rows without a cell are zero; a bad sample's, and all after a wait that ran out, NaN.
        const float scale = width > 0 ? 1.f / sum : 0.f;
        const bool broken = !ok || !good;
        T* out = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.N + i) * a.Hq + h) * a.d;
        T* out_lo = a.out_lo ? static_cast<T*>(a.out_lo) + ((static_cast<int64_t>(b) * a.N + i) * a.Hq + h) * a.d : nullptr;
        for (int c = 0; c < a.d; c += 32) {
            float v[32];
            if (jb_w > ja_w && ok) {
                uint32_t o[32];
                tmem_ld32(to + c, o);
                wait_ld();
                settle(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = width > 0 ? __uint_as_float(o[e]) * scale : 0.f;
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0.f;
            }
            if (broken) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __int_as_float(0x7fc00000);
            }
            if (i < a.N) store_row32<T>(out, out_lo, v, c, a.d);
        }
        if (i < a.N && a.lse)
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
    static std::mutex mu;
    static bool set[128] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 128) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!set[dev]) {
            e = cudaFuncSetAttribute(attend_tc_kernel<T, DPAD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::BYTES);
            if (e != cudaSuccess) return e;
            set[dev] = true;
        }
    }
    f.tiles = static_cast<int>((f.a.N + kTile * NT - 1) / (kTile * NT));
    const int64_t grid = static_cast<int64_t>(f.a.B) * f.a.Hq * f.tiles;
    attend_tc_kernel<T, DPAD, NT><<<static_cast<unsigned>(grid), G::THREADS, G::BYTES, s>>>(mq, mk, mv, f);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward_t(const AttnArgs& a, cudaStream_t s)
{
    CUtensorMap mq, mk, mv;
    constexpr bool half = std::is_same<T, __half>::value;
    if (!attention_tile_map(&mq, half, a.q, a.qs, a.B, a.N, a.Hq, a.d, kTile) ||
        !attention_tile_map(&mk, half, a.k, a.ks, a.B, a.M, a.Hkv, a.d, kTile) ||
        !attention_tile_map(&mv, half, a.v, a.vs, a.B, a.M, a.Hkv, a.d, kTile))
        return cudaErrorInvalidValue;
    FwdArgs f{};
    f.a = a;
    f.timeout_ns = static_cast<uint64_t>(wait_timeout_s() * 1e9);
    f.dn = (a.d + 15) / 16 * 16;
    f.negative = a.scale_log2 < 0;
    f.a.scale_log2 = fmaxf(fabsf(a.scale_log2), 1e-30f);  // a scale of zero: all scores equal
    if (a.d <= 64) return launch_forward<T, 64, 1>(f, mq, mk, mv, s);
    return launch_forward<T, 128, 2>(f, mq, mk, mv, s);
}

}  // namespace

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
