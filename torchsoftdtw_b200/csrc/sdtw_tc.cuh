// Thin wrappers of the sm_100a asynchronous machinery that the attention kernels share: mbarriers with bounded
// waits, TMA loads, tcgen05 products of 16-bit operands (fp32 accumulators in tensor memory), descriptors.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "sdtw_sequence.cuh"

namespace sdtw {
namespace tc {

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.b32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}

// The bound of every wait of a CTA, and the word that ends them all when one ran out.
struct Bound {
    uint64_t timeout_ns;
    volatile int* abort;  // shared memory
    uint32_t* err;
};

// Up to 1024 tries (each of which the hardware suspends for a while). A wait for a phase that is already complete costs 44
// cycles as a single try, 85 with the vote and this loop behind it, 216 as a loop in C++: the MMA warps make half a dozen a tile.
__device__ __forceinline__ bool mbar_spin(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p, q; .reg .u32 n; mov.u32 n, 0;\n"
        "AGAIN_%=: mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "@p bra DONE_%=;\n"
        "add.u32 n, n, 1; setp.lt.u32 q, n, 1024;\n"
        "@q bra AGAIN_%=;\n"
        "DONE_%=: selp.b32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// A wait that has not ended in mbar_spin: goes on until the phase completes, the time runs out or another role gives up.
static __device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity, Bound w)
{
    const uint64_t t0 = global_ns();
    bool mine = false;
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 64 && !mine; ++i) mine = mbar_try_wait(bar, parity);
        __syncwarp();
        if (__all_sync(kFull, mine)) return true;
        const bool late = global_ns() - t0 > w.timeout_ns;
        if (__any_sync(kFull, late || *w.abort)) {
            if ((threadIdx.x & 31) == 0 && !*w.abort) {
                *w.abort = 1;
                atomicOr(w.err, kErrTimeout);
            }
            return false;
        }
    }
}

// Waits, as a whole warp, for the phase with the given parity. False, for all its lanes, when it ran out of time, or
// another role of the CTA did.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Bound& w)
{
    if (__all_sync(kFull, mbar_try_wait(bar, parity))) return true;
    if (__all_sync(kFull, mbar_spin(bar, parity))) return true;
    return mbar_wait_long(bar, parity, w);
}
// The same wait for one's own operations in flight, which goes on after an abort.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity, uint64_t timeout_ns)
{
    if (mbar_spin(bar, parity)) return;
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bar, parity) && global_ns() - t0 <= timeout_ns) {
    }
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The warp that issues products runs them as one: its control flow and descriptors stay uniform, and only the
// instructions themselves are for its leader. (Inside a branch of one lane each product cost about 110 cycles of
// operand moves, against the 64 that the tensor core takes for it.)
__device__ __forceinline__ uint32_t elect_leader()
{
    uint32_t is;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.b32 %0, 1, 0, p; }" : "=r"(is));
    return is;
}
// Arrives on the barrier when every product issued by the leader so far has completed.
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t leader)
{
    asm volatile(
        "{ .reg .pred q; setp.ne.b32 q, %1, 0; "
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar),
        "r"(leader)
        : "memory");
}

// Instruction descriptor: fp32 accumulators, 16-bit operands (both bf16 or both fp16), A 128 rows, B n columns; b_mn:
// B lies with its columns (n) contiguous in memory instead of its K.
template <typename T>
__device__ __forceinline__ constexpr uint32_t mma_idesc(int n, bool b_mn)
{
    constexpr uint32_t t = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(128 >> 4) << 24);
}

// Operand descriptors of a tile that TMA wrote with the 128-byte swizzle: 64 elements (128 bytes) a row, rows
// 128 bytes apart, 8-row groups 1024 bytes apart; wider tiles are blocks of 64 columns, `block` bytes apart.
// K-major: rows are the operand's rows (or columns of B), K runs along the 128 bytes.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr)
{
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// A descriptor `bytes` further on (a tile lies below 256 KB, so its address field takes the sum).
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
// MN-major: the tile's rows are K, its 64-column blocks the operand's columns.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t block)
{
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// d += a b (accumulate) or d = a b: A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t leader)
{
    asm volatile(
        "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; "
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(leader)
        : "memory");
}
// The same with A in tensor memory: lane = row, each 32-bit column two neighbouring K.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t leader)
{
    asm volatile(
        "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; "
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// 32 consecutive columns of this thread's lane. Nothing is waited for.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// The values that tcgen05.ld delivers exist only after wait_ld: this keeps their uses below it.
template <int N>
__device__ __forceinline__ void settle(uint32_t (&r)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

}  // namespace tc
}  // namespace sdtw
