// What the attention kernels on warp-level mma share: fragments, the split of float32 operands, and row copies of any
// alignment.
//
// Fragments (one m16n8 accumulator c: rows lane / 4 and + 8, columns 2 (lane % 4) and + 1): 16-bit operands by m16n8k16,
// float32 as three TF32 products m16n8k8 of an 11-bit head and tail (x = head + tail to 2^-23; tail.tail is dropped). The
// matrix pipe's adder cuts off where an add in 32 bits rounds, an error of one sign for each instruction that a sum goes
// through. So at most four head products follow one another before their sum is added to the total by an ordinary add, and
// the tails' products have a sum of their own, 2^-11 of the heads'.
#pragma once

#include <type_traits>

#include "sdtw_attention.h"

namespace sdtw {

__device__ __forceinline__ float tf32(float x)
{
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return __uint_as_float(r);
}
__device__ __forceinline__ void split2(float x, uint32_t& head, uint32_t& tail)
{
    const float h = tf32(x);
    head = __float_as_uint(h);
    tail = __float_as_uint(tf32(x - h));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int NB>
__device__ __forceinline__ void add(float (&c)[NB][4], const float (&x)[NB][4])
{
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i][e] += x[i][e];
}
template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// c[x] += A B^T for the NB 8-row groups of B: A 16 rows, B 8 NB rows, both row-major of pitch LD in shared memory, K over their
// DPAD features.
template <typename T, int DPAD, int LD, int NB>
__device__ __forceinline__ void product_rows(float (&c)[NB][4], const T* A, const T* B, int lane)
{
    if constexpr (sizeof(T) == 2) {
        static_assert(NB % 2 == 0, "16 rows of B at a time");
        const uint32_t a_at = smem_addr(A) + 2 * ((lane & 15) * LD + (lane >> 4) * 8);
        const uint32_t b_at = smem_addr(B) + 2 * (((lane & 7) + ((lane >> 4) & 1) * 8) * LD + ((lane >> 3) & 1) * 8);
#pragma unroll
        for (int k = 0; k < DPAD; k += 16) {
            uint32_t a[4];
            ldmatrix4(a_at + 2 * k, a);
#pragma unroll
            for (int x = 0; x < NB / 2; ++x) {
                uint32_t b[4];
                ldmatrix4(b_at + 2 * (16 * x * LD + k), b);
                mma_16<T>(c[2 * x], a, b[0], b[1]);
                mma_16<T>(c[2 * x + 1], a, b[2], b[3]);
            }
        }
    } else {
        const float* ar = A + (lane >> 2) * LD + (lane & 3);
        const float* br = B + (lane >> 2) * LD + (lane & 3);
        float tails[NB][4] = {};
#pragma unroll 1
        for (int k0 = 0; k0 < DPAD; k0 += 32) {
            float heads[NB][4] = {};
#pragma unroll
            for (int k = k0; k < k0 + 32; k += 8) {
                uint32_t ah[4], al[4];
                split2(ar[k], ah[0], al[0]);
                split2(ar[8 * LD + k], ah[1], al[1]);
                split2(ar[k + 4], ah[2], al[2]);
                split2(ar[8 * LD + k + 4], ah[3], al[3]);
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    uint32_t bh[2], bl[2];
                    split2(br[8 * x * LD + k], bh[0], bl[0]);
                    split2(br[8 * x * LD + k + 4], bh[1], bl[1]);
                    mma_tf32(tails[x], al, bh[0], bh[1]);
                    mma_tf32(heads[x], ah, bh[0], bh[1]);
                    mma_tf32(tails[x], ah, bl[0], bl[1]);
                }
            }
            add(c, heads);
        }
        add(c, tails);
    }
}

// o += S B: S 16 x 8 NB in accumulator layout, B 8 NB rows of DPAD features, row-major of pitch LD in shared memory.
template <typename T, int DPAD, int LD, int NB>
__device__ __forceinline__ void product_columns(float (&o)[DPAD / 8][4], const float (&s)[NB][4], const T* B, int lane)
{
    if constexpr (sizeof(T) == 2) {
        const uint32_t b_at = smem_addr(B) + 2 * (((lane & 7) + ((lane >> 3) & 1) * 8) * LD + ((lane >> 4) & 1) * 8);
#pragma unroll
        for (int x = 0; x < NB / 2; ++x) {
            const uint32_t a[4] = {pack2(s[2 * x][0], s[2 * x][1], T()), pack2(s[2 * x][2], s[2 * x][3], T()),
                                   pack2(s[2 * x + 1][0], s[2 * x + 1][1], T()), pack2(s[2 * x + 1][2], s[2 * x + 1][3], T())};
#pragma unroll
            for (int y = 0; y < DPAD / 16; ++y) {
                uint32_t b[4];
                ldmatrix4t(b_at + 2 * (16 * x * LD + 16 * y), b);
                mma_16<T>(o[2 * y], a, b[0], b[1]);
                mma_16<T>(o[2 * y + 1], a, b[2], b[3]);
            }
        }
    } else {
        // The accumulator's columns 2t, 2t + 1 serve as the operand's K = t, t + 4; B's rows are taken in that order.
        const float* br = B + 2 * (lane & 3) * LD + (lane >> 2);
        static_assert(NB <= 4, "four head products a sum");
        uint32_t ah[NB][4], al[NB][4];
#pragma unroll
        for (int x = 0; x < NB; ++x) {
            split2(s[x][0], ah[x][0], al[x][0]);
            split2(s[x][2], ah[x][1], al[x][1]);
            split2(s[x][1], ah[x][2], al[x][2]);
            split2(s[x][3], ah[x][3], al[x][3]);
        }
#pragma unroll
        for (int y = 0; y < DPAD / 8; ++y) {
            float heads[4] = {}, tails[4] = {};
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                uint32_t bh[2], bl[2];
                split2(br[8 * x * LD + 8 * y], bh[0], bl[0]);
                split2(br[(8 * x + 1) * LD + 8 * y], bh[1], bl[1]);
                mma_tf32(tails, al[x], bh[0], bh[1]);
                mma_tf32(heads, ah[x], bh[0], bh[1]);
                mma_tf32(tails, ah[x], bl[0], bl[1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[y][e] += heads[e] + tails[e];
        }
    }
}

// One 16-byte unit of a row (features f ..) from global to shared memory, in pieces of VB bytes; features from d on are
// not touched (they were cleared), nor read. A row that is not `on` becomes zero.
template <typename T, int VB>
__device__ __forceinline__ void copy_unit(T* dst, const T* src, int f, int d, bool on)
{
    constexpr int E = VB / static_cast<int>(sizeof(T)), UNIT = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int e = 0; e < UNIT; e += E) {
        if (f + e >= d) break;
        if constexpr (VB == 16)
            cp_async_16(dst, src, on ? 16 : 0);
        else if constexpr (VB == 4)
            cp_async_4(dst + e, src + e, on ? 4 : 0);
        else
            dst[e] = on ? src[e] : from_f<T>(0.f);
    }
}

// The bits of an operand's address and steps, in bytes; copy_bytes: the largest piece that everything starts on a multiple of.
template <typename T>
inline uintptr_t step_bits(const void* p, const Strides& s)
{
    return reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>((s.b | s.n | s.h) * static_cast<int64_t>(sizeof(T)));
}
inline int copy_bytes(uintptr_t bits) { return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 2); }

}  // namespace sdtw
