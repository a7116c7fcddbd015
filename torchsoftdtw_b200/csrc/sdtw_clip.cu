// The global norm of many tensors, and their clipping by it:
//   norm = (sum over all entries of g^2)^(1/2)   or   max |g|;   out = g * min(1, max_norm / (norm + 1e-6)).
//
// Bound by memory: one read for the norm, one read and one write for the scaling (no read or write where the
// factor is one and the tensors are scaled in place). Two launches: the first leaves one partial result per
// CTA, the second combines the partials in every CTA (in one fixed order, so each run and each CTA gets the
// same bits) and scales. Tensors are cut into chunks of 64 KB, or less where there would be fewer than four chunks a
// CTA; CTA c takes chunks c, c + grid, and the second launch walks them backwards, so that what the first one read last is
// still in L2: 252 million bf16 (504 MB) 252 us in place, 6.0 TB/s of its 1.51 GB; 231 us is a copy's rate for them.
// Few small tensors are bound by the two launches: 25 tensors, 0.4 MB, 19 us a call with the host's part.
#include <cmath>
#include <cstring>

#include "sdtw_sequence.cuh"

namespace sdtw {
namespace {

constexpr int kThreads = 512;
constexpr int kMinChunk = 8192, kMaxChunk = 65536;  // bytes
constexpr int kCtasPerSm = 3;
constexpr int kMaxCtas = 1024;       // partial results per launch
constexpr int kSmallCap = 64;        // tensors per launch: the table is a kernel argument (32 KB at most)
constexpr int kLargeCap = 960;
constexpr double kClipEps = 1e-6;

struct Entry {
    const void* src;
    void* dst;
    int64_t n;
    int32_t first_chunk;
    int32_t dtype;
};

template <int CAP>
struct Table {
    Entry e[CAP];
    int32_t count;
    int32_t chunks;
    int32_t wide;  // some tensor is float64: every square is formed in 64 bits, its range extended
    int32_t kind;  // 0: Euclidean, 1: largest magnitude
    int32_t chunk_bytes;
};

__host__ __device__ __forceinline__ int chunk_entries(int bytes, int dtype)
{
    return bytes >> (dtype == SDTW_F64 ? 3 : (dtype == SDTW_F32 ? 2 : 1));
}

template <int CAP>
__device__ __forceinline__ int find_entry(const Table<CAP>& t, int chunk)
{
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first_chunk <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double wide_of(float x) { return static_cast<double>(x); }
__device__ __forceinline__ double wide_of(double x) { return x; }
__device__ __forceinline__ double wide_of(__half x) { return static_cast<double>(__half2float(x)); }
__device__ __forceinline__ double wide_of(__nv_bfloat16 x) { return static_cast<double>(__bfloat162float(x)); }

// f(entry, j) for every entry of [p, p + n) that this thread owns, j its place in its 16-byte access: four
// accesses in flight when p is aligned, single entries (j = 0) otherwise and for the tail.
template <typename T, typename F>
__device__ __forceinline__ void for_entries(const T* p, int n, F f)
{
    constexpr int V = 16 / sizeof(T);
    int i = 0;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const Vec<T, V>* pv = reinterpret_cast<const Vec<T, V>*>(p);
        const int nv = n / V;
        int k = threadIdx.x;
        for (; k + 3 * kThreads < nv; k += 4 * kThreads) {
            Vec<T, V> v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = pv[k + u * kThreads];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) f(v[u].e[j], j);
        }
        for (; k < nv; k += kThreads) {
            const Vec<T, V> v = pv[k];
#pragma unroll
            for (int j = 0; j < V; ++j) f(v.e[j], j);
        }
        i = nv * V;
    }
    for (i += threadIdx.x; i < n; i += kThreads) f(p[i], 0);
}

// A sum of squares whose float64 entries may square out of their range: entries above 2^400 enter `big` scaled
// by 2^-600, entries below 2^-400 `small` scaled by 2^600, all others `mid`. Scaled, the largest entry squares to 2^848, the
// smallest subnormal one to 2^-948, and those next to the borders to 2^-400 and 2^400.
struct Squares {
    double mid, big, small;
};
constexpr double kUp = 0x1p600, kDown = 0x1p-600;

__device__ __forceinline__ double norm_of(const Squares& q)
{
    if (q.big > 0.0) return sqrt(q.big + q.mid * kDown * kDown) * kUp;
    if (q.small > 0.0 && q.mid < 0x1p-700) return sqrt(q.small + q.mid * kUp * kUp) * kDown;
    return sqrt(q.mid);
}

// Adds this thread's part of a chunk's sum of squares. Up to 64 squares a thread are added in 32 bits (relative
// error below 64 * 2^-24, far below it in the sum over threads); a sum that is not finite or so small that
// squares may have underflowed is formed again in 64 bits (the chunk is in the caches by then).
template <typename T>
__device__ __forceinline__ void chunk_squares(const T* p, int n, bool wide, Squares& q)
{
    if constexpr (sizeof(T) < 8) {
        if (!wide) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            float big = 0.f;
            for_entries(p, n, [&](T x, int j) {
                const float v = to_f(x);
                s[j & 3] = fmaf(v, v, s[j & 3]);
                big = fmaxf(big, fabsf(v));
            });
            const float t = (s[0] + s[1]) + (s[2] + s[3]);
            if (t < 1e36f && (t > 1e-24f || big == 0.f)) {
                q.mid += static_cast<double>(t);
                return;
            }
        }
    }
    for_entries(p, n, [&](T x, int) {
        const double v = wide_of(x);
        if constexpr (sizeof(T) == 8) {
            const double m = fabs(v);
            if (m > 0x1p400) {
                q.big = fma(v * kDown, v * kDown, q.big);
                return;
            }
            if (m < 0x1p-400) {
                q.small = fma(v * kUp, v * kUp, q.small);
                return;
            }
        }
        q.mid = fma(v, v, q.mid);
    });
}

// The largest magnitude as the bits of a double: for non-negative doubles the order of the bits is that of
// the values, and every NaN lies above infinity, so one integer maximum carries NaN through.
template <typename T>
__device__ __forceinline__ unsigned long long chunk_largest(const T* p, int n)
{
    if constexpr (sizeof(T) == 8) {
        unsigned long long m = 0;
        for_entries(p, n, [&](T x, int) { m = max(m, static_cast<unsigned long long>(__double_as_longlong(fabs(x)))); });
        return m;
    } else {
        unsigned m = 0;
        for_entries(p, n, [&](T x, int) { m = max(m, __float_as_uint(to_f(x)) & 0x7fffffffu); });
        return static_cast<unsigned long long>(__double_as_longlong(static_cast<double>(__uint_as_float(m))));
    }
}

struct Sum {
    static __device__ __forceinline__ double join(double a, double b) { return a + b; }
};
struct Largest {
    static __device__ __forceinline__ double join(double a, double b)
    {
        return __longlong_as_double(static_cast<long long>(
            max(static_cast<unsigned long long>(__double_as_longlong(a)),
                static_cast<unsigned long long>(__double_as_longlong(b)))));
    }
};

// The same result in every thread, joined in a fixed order.
template <typename OP>
__device__ double block_join(double v, double* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = OP::join(v, __shfl_xor_sync(kFull, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) t = OP::join(t, red[w]);
    __syncthreads();  // red is used again
    return t;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) clip_partials_kernel(const __grid_constant__ Table<CAP> t,
                                                                             Squares* partials)
{
    __shared__ double red[kThreads / 32];
    Squares acc = {0.0, 0.0, 0.0};
    unsigned long long top = 0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Entry& e = t.e[find_entry(t, c)];
        const int chunk = chunk_entries(t.chunk_bytes, e.dtype);
        const int64_t at = static_cast<int64_t>(c - e.first_chunk) * chunk;
        const int n = static_cast<int>(min(static_cast<int64_t>(chunk), e.n - at));
        const bool wide = t.wide != 0;
        if (t.kind == 0) {
            switch (e.dtype) {
                case SDTW_F32: chunk_squares(static_cast<const float*>(e.src) + at, n, wide, acc); break;
                case SDTW_F64: chunk_squares(static_cast<const double*>(e.src) + at, n, wide, acc); break;
                case SDTW_F16: chunk_squares(static_cast<const __half*>(e.src) + at, n, wide, acc); break;
                default: chunk_squares(static_cast<const __nv_bfloat16*>(e.src) + at, n, wide, acc); break;
            }
        } else {
            switch (e.dtype) {
                case SDTW_F32: top = max(top, chunk_largest(static_cast<const float*>(e.src) + at, n)); break;
                case SDTW_F64: top = max(top, chunk_largest(static_cast<const double*>(e.src) + at, n)); break;
                case SDTW_F16: top = max(top, chunk_largest(static_cast<const __half*>(e.src) + at, n)); break;
                default: top = max(top, chunk_largest(static_cast<const __nv_bfloat16*>(e.src) + at, n)); break;
            }
        }
    }
    if (t.kind != 0) {
        const double v = block_join<Largest>(__longlong_as_double(static_cast<long long>(top)), red);
        if (threadIdx.x == 0) partials[blockIdx.x].mid = v;
        return;
    }
    Squares q;
    q.mid = block_join<Sum>(acc.mid, red);
    q.big = t.wide ? block_join<Sum>(acc.big, red) : 0.0;
    q.small = t.wide ? block_join<Sum>(acc.small, red) : 0.0;
    if (threadIdx.x == 0) partials[blockIdx.x] = q;
}

template <typename T, typename C>
__device__ __forceinline__ T scaled(T x, C c)
{
    if constexpr (sizeof(T) == 8)
        return x * c;
    else
        return from_f<T>(to_f(x) * static_cast<float>(c));
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* src, T* dst, int n, double coef)
{
    constexpr int V = 16 / sizeof(T);
    int i = 0;
    if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0) {
        const Vec<T, V>* s = reinterpret_cast<const Vec<T, V>*>(src);
        uint4* d = reinterpret_cast<uint4*>(dst);
        const int nv = n / V;
        int k = threadIdx.x;
        auto put = [&](const Vec<T, V>& v, int at) {
            union {
                Vec<T, V> o;
                uint4 u;
            } w;
#pragma unroll
            for (int j = 0; j < V; ++j) w.o.e[j] = scaled(v.e[j], coef);
            __stcs(d + at, w.u);
        };
        for (; k + 3 * kThreads < nv; k += 4 * kThreads) {
            Vec<T, V> v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = s[k + u * kThreads];
#pragma unroll
            for (int u = 0; u < 4; ++u) put(v[u], k + u * kThreads);
        }
        for (; k < nv; k += kThreads) put(s[k], k);
        i = nv * V;
    }
    for (i += threadIdx.x; i < n; i += kThreads) dst[i] = scaled(src[i], coef);
}

struct ScaleArgs {
    const Squares* partials;
    int32_t partial_count;
    int32_t norm_f64;
    double max_norm;
    void* norm_out;
};

template <int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) clip_scale_kernel(const __grid_constant__ Table<CAP> t,
                                                                          const ScaleArgs a)
{
    __shared__ double red[kThreads / 32];
    Squares q = {0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < a.partial_count; i += kThreads) {
        const Squares p = a.partials[i];
        q.mid = t.kind == 0 ? q.mid + p.mid : Largest::join(q.mid, p.mid);
        q.big += p.big;
        q.small += p.small;
    }
    double norm;
    if (t.kind == 0) {
        q.mid = block_join<Sum>(q.mid, red);
        if (t.wide) {
            q.big = block_join<Sum>(q.big, red);
            q.small = block_join<Sum>(q.small, red);
        }
        norm = norm_of(q);
    } else {
        norm = block_join<Largest>(q.mid, red);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (a.norm_f64)
            *static_cast<double*>(a.norm_out) = norm;
        else
            *static_cast<float*>(a.norm_out) = static_cast<float>(norm);
    }
    const double ratio = a.max_norm / (norm + kClipEps);
    const double coef = ratio > 1.0 ? 1.0 : ratio;  // a NaN stays
    for (int c = t.chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= static_cast<int>(gridDim.x)) {
        const Entry& e = t.e[find_entry(t, c)];
        if (coef == 1.0 && e.src == e.dst) continue;
        const int chunk = chunk_entries(t.chunk_bytes, e.dtype);
        const int64_t at = static_cast<int64_t>(c - e.first_chunk) * chunk;
        const int n = static_cast<int>(min(static_cast<int64_t>(chunk), e.n - at));
        switch (e.dtype) {
            case SDTW_F32:
                scale_chunk(static_cast<const float*>(e.src) + at, static_cast<float*>(e.dst) + at, n, coef);
                break;
            case SDTW_F64:
                scale_chunk(static_cast<const double*>(e.src) + at, static_cast<double*>(e.dst) + at, n, coef);
                break;
            case SDTW_F16:
                scale_chunk(static_cast<const __half*>(e.src) + at, static_cast<__half*>(e.dst) + at, n, coef);
                break;
            default:
                scale_chunk(static_cast<const __nv_bfloat16*>(e.src) + at, static_cast<__nv_bfloat16*>(e.dst) + at, n,
                            coef);
                break;
        }
    }
}

int clip_grid(int chunks, int sms) { return chunks < sms * kCtasPerSm ? chunks : sms * kCtasPerSm; }

template <int CAP>
sdtw_status clip_run(const sdtw_tensor_ref* refs, int64_t count, int kind, bool wide, bool scale, double max_norm,
                     void* norm, int norm_f64, Squares* partials, int sms, cudaStream_t s)
{
    // Tables of CAP tensors, non-empty ones only; the same cut in both passes.
    Table<CAP> t;
    t.wide = wide;
    t.kind = kind;
    int64_t bytes = 0;
    for (int64_t i = 0; i < count; ++i) bytes += refs[i].numel * static_cast<int64_t>(dtype_size(refs[i].dtype));
    t.chunk_bytes = kMaxChunk;
    while (t.chunk_bytes > kMinChunk && bytes / t.chunk_bytes < 4 * sms * kCtasPerSm) t.chunk_bytes /= 2;
    int64_t at = 0;
    auto fill = [&]() -> sdtw_status {
        t.count = 0;
        t.chunks = 0;
        for (; at < count && t.count < CAP; ++at) {
            const int64_t n = refs[at].numel;
            if (n == 0) continue;
            const int64_t chunk = chunk_entries(t.chunk_bytes, refs[at].dtype), chunks = (n + chunk - 1) / chunk;
            if (chunks > (1 << 28) || t.chunks > (1 << 28)) return SDTW_EINVAL;
            t.e[t.count++] = {refs[at].src, refs[at].dst, n, t.chunks, refs[at].dtype};
            t.chunks += static_cast<int32_t>(chunks);
        }
        return SDTW_OK;
    };
    int64_t total = 0;
    while (at < count) {
        const sdtw_status st = fill();
        if (st != SDTW_OK) return st;
        if (t.chunks == 0) break;
        const int grid = clip_grid(t.chunks, sms);
        clip_partials_kernel<CAP><<<grid, kThreads, 0, s>>>(t, partials + total);
        count_launch();
        total += grid;
    }
    ScaleArgs a{partials, static_cast<int32_t>(total), norm_f64, max_norm, norm};
    at = 0;
    bool first = true;
    while (first || (scale && at < count)) {
        t.count = 0;
        t.chunks = 0;
        if (scale) {
            const sdtw_status st = fill();
            if (st != SDTW_OK) return st;
        }
        if (!first && t.chunks == 0) break;
        clip_scale_kernel<CAP><<<t.chunks ? clip_grid(t.chunks, sms) : 1, kThreads, 0, s>>>(t, a);
        count_launch();
        first = false;
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SDTW_OK : static_cast<sdtw_status>(e);
}

sdtw_status clip_any(const sdtw_tensor_ref* refs, int64_t count, int kind, bool scale, double max_norm, void* norm,
                     int norm_f64, void* workspace, size_t workspace_bytes, void* stream)
{
    if (count < 0 || (count > 0 && refs == nullptr) || norm == nullptr || (kind != SDTW_NORM_L2 && kind != SDTW_NORM_MAX))
        return SDTW_EINVAL;
    if (scale && !(max_norm >= 0)) return SDTW_EINVAL;
    bool wide = false;
    for (int64_t i = 0; i < count; ++i) {
        const sdtw_tensor_ref& r = refs[i];
        if (r.numel < 0 || (r.numel > 0 && (r.src == nullptr || (scale && r.dst == nullptr)))) return SDTW_EINVAL;
        if (r.dtype < SDTW_F32 || r.dtype > SDTW_BF16) return SDTW_EDTYPE;
        wide = wide || r.dtype == SDTW_F64;
    }
    if (workspace == nullptr || workspace_bytes < sdtw_clip_workspace_bytes(count)) return SDTW_EWORKSPACE;
    int dev = 0, sms = 0;
    const cudaError_t e = current_sms(dev, sms);
    if (e != cudaSuccess) return static_cast<sdtw_status>(e);
    if (sms * kCtasPerSm > kMaxCtas) sms = kMaxCtas / kCtasPerSm;
    Squares* partials = static_cast<Squares*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return count <= kSmallCap ? clip_run<kSmallCap>(refs, count, kind, wide, scale, max_norm, norm, norm_f64, partials, sms, s)
                              : clip_run<kLargeCap>(refs, count, kind, wide, scale, max_norm, norm, norm_f64, partials, sms, s);
}

}  // namespace
}  // namespace sdtw

extern "C" {

size_t sdtw_clip_workspace_bytes(int64_t count)
{
    using namespace sdtw;
    const int64_t launches = count <= kSmallCap ? 1 : (count + kLargeCap - 1) / kLargeCap;
    return static_cast<size_t>(launches) * kMaxCtas * sizeof(Squares);
}

sdtw_status sdtw_global_norm(const sdtw_tensor_ref* tensors, int64_t count, int norm_kind, void* norm, int norm_f64,
                             void* workspace, size_t workspace_bytes, void* stream)
{
    return sdtw::clip_any(tensors, count, norm_kind, false, 0.0, norm, norm_f64, workspace, workspace_bytes, stream);
}

sdtw_status sdtw_clip_grads(const sdtw_tensor_ref* tensors, int64_t count, int norm_kind, double max_norm, void* norm,
                            int norm_f64, void* workspace, size_t workspace_bytes, void* stream)
{
    return sdtw::clip_any(tensors, count, norm_kind, true, max_norm, norm, norm_f64, workspace, workspace_bytes, stream);
}

}  // extern "C"
