// PyTorch operator layer of the sequence-model operators beside the loss: torchsoftdtw_b200::cross_attention (with
// attention / attention_backward below autograd), norm_rotate / norm_rotate_backward, global_norm / clip_grads. It
// checks arguments, allocates outputs and workspaces, and forwards every call to the C ABI (include/sdtw_b200.h).
// Autograd is in C++: at these kernels' times, a training step through Python functions would be bound by the host
// (about 100 us a step against 45 us of kernels at 32 x 512 x 8 x 64).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "sdtw_b200.h"
#include "torch_ops.h"

namespace {

using at::Tensor;
using sdtw_ops::check_status;
using sdtw_ops::error_word;
using sdtw_ops::maybe_sync_check;
using OptTensor = std::optional<Tensor>;

sdtw_dtype code_of(at::ScalarType st)
{
    switch (st) {
        case at::kFloat: return SDTW_F32;
        case at::kDouble: return SDTW_F64;
        case at::kHalf: return SDTW_F16;
        default: return SDTW_BF16;
    }
}

// Numbers reach messages through std::to_string: streaming one from this library ends the process under the
// C++ runtime that this Python loads.
template <typename T>
std::string num(T x)
{
    return std::to_string(x);
}

// "[2, 3]", for messages.
std::string shape_of(const Tensor& t)
{
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i > 0 ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

void cuda_tensor(const Tensor& t)
{
    TORCH_CHECK(t.is_cuda(), "torchsoftdtw_b200 runs on CUDA devices only (sm_100); got a tensor on ", t.device());
}

void float_type(const Tensor& t, const char* name)
{
    const auto st = t.scalar_type();
    TORCH_CHECK(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, name,
                " must be float16, bfloat16 or float32, got ", st);
}

void lengths_check(const OptTensor& l, int64_t B, const Tensor& like, const char* name)
{
    if (!l) return;
    TORCH_CHECK(l->dim() == 1 && l->size(0) == B, name, " must have shape (", num(B), ",), got ", shape_of(*l));
    TORCH_CHECK(l->scalar_type() == at::kInt || l->scalar_type() == at::kLong, name, " must be int32 or int64");
    TORCH_CHECK(l->device() == like.device(), name, " must be on ", like.device(), ", got ", l->device());
}

// t with neighbouring features, as the kernels read it: t itself, or a contiguous copy.
Tensor feature_rows(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// t as the tensor-core kernels read it (16-byte steps in every dimension), copied where that is all it lacks: their
// time is several times less than that of the kernels for any layout, even with the copy.
Tensor tensor_core_rows(const Tensor& t)
{
    const Tensor r = feature_rows(t);
    if (r.scalar_type() == at::kFloat || r.size(-1) % 8 != 0) return r;
    bool fits = reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fits = fits && (r.size(i) == 1 || (r.stride(i) > 0 && r.stride(i) % 8 == 0));
    if (fits) return r;
    return r.is_contiguous() ? r.clone(at::MemoryFormat::Contiguous) : r.contiguous();
}

Tensor workspace_of(size_t bytes, const Tensor& like)
{
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ---------------------------------------------------------------------------------------------------
// Cross attention
// ---------------------------------------------------------------------------------------------------
void attention_checks(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lx, const OptTensor& ly,
                      double scale)
{
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                "q must be 4D (B, N, Hq, d), k and v 4D (B, M, Hkv, d)");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape, got ", shape_of(k), " and ", shape_of(v));
    TORCH_CHECK(q.size(0) == k.size(0), "Batch size mismatch between q and k");
    TORCH_CHECK(q.size(3) == k.size(3), "q and k must have the same head dimension");
    TORCH_CHECK(q.size(3) >= 1 && q.size(3) <= 128, "the head dimension must lie in [1, 128], got ", num(q.size(3)));
    TORCH_CHECK(k.size(2) >= 1 && q.size(2) >= 1 && q.size(2) % k.size(2) == 0,
                "the query heads must be a positive multiple of the key heads, got ", num(q.size(2)), " and ",
                num(k.size(2)));
    TORCH_CHECK(std::isfinite(scale), "scale must be finite");
    float_type(q, "q");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                "q, k and v must have the same dtype");
    cuda_tensor(q);
    TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "q, k and v must be on the same device");
    lengths_check(lx, q.size(0), q, "lengths_x");
    lengths_check(ly, q.size(0), q, "lengths_y");
}

struct AttentionCall {
    sdtw_attention_problem p{};
    Tensor q, k, v, lx, ly;  // what p points into
};

// tensor_core: the call is one that the tensor-core kernels take (a decoded token's cache, for one, is never copied).
void fill_attention(AttentionCall& c, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_x,
                    const OptTensor& lengths_y, int64_t bandwidth, double scale, bool tensor_core)
{
    c.q = tensor_core ? tensor_core_rows(q) : feature_rows(q);
    c.k = tensor_core ? tensor_core_rows(k) : feature_rows(k);
    c.v = tensor_core ? tensor_core_rows(v) : feature_rows(v);
    sdtw_attention_problem& p = c.p;
    p.dtype = code_of(q.scalar_type());
    // Both lengths are read with one element type.
    const bool wide = (lengths_x && lengths_x->scalar_type() == at::kLong) ||
                      (lengths_y && lengths_y->scalar_type() == at::kLong);
    const auto as = [&](const OptTensor& l) {
        return l ? l->to(wide ? at::kLong : at::kInt).contiguous() : Tensor();
    };
    c.lx = as(lengths_x);
    c.ly = as(lengths_y);
    p.lengths_int32 = !wide;
    p.lengths_x = c.lx.defined() ? c.lx.data_ptr() : nullptr;
    p.lengths_y = c.ly.defined() ? c.ly.data_ptr() : nullptr;
    p.q = c.q.data_ptr();
    p.k = c.k.data_ptr();
    p.v = c.v.data_ptr();
    for (int i = 0; i < 3; ++i) {
        p.q_stride[i] = c.q.stride(i);
        p.k_stride[i] = c.k.stride(i);
        p.v_stride[i] = c.v.stride(i);
    }
    p.B = q.size(0);
    p.N = q.size(1);
    p.M = k.size(1);
    p.Hq = q.size(2);
    p.Hkv = k.size(2);
    p.d = q.size(3);
    p.bandwidth = bandwidth;
    p.scale = scale;
    p.err_word = error_word(q);
}

// The forward; with `grad`, also what the backward needs: out_lo (16-bit types) and lse.
Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_x,
                         const OptTensor& lengths_y, int64_t bandwidth, double scale, bool grad, Tensor* out_lo, Tensor* lse)
{
    attention_checks(q, k, v, lengths_x, lengths_y, scale);
    const c10::cuda::CUDAGuard guard(q.device());
    AttentionCall c;
    fill_attention(c, q, k, v, lengths_x, lengths_y, bandwidth, scale, q.size(1) * (q.size(2) / k.size(2)) > 64);
    const Tensor out = at::empty({c.p.B, c.p.N, c.p.Hq, c.p.d}, q.options());
    void* lo_ptr = nullptr;
    float* lse_ptr = nullptr;
    if (grad) {
        *lse = at::empty({c.p.B, c.p.Hq, c.p.N}, q.options().dtype(at::kFloat));
        lse_ptr = lse->data_ptr<float>();
        const bool lo = q.scalar_type() != at::kFloat;
        *out_lo = lo ? at::empty({c.p.B, c.p.N, c.p.Hq, c.p.d}, q.options()) : at::empty({0}, q.options());
        if (lo) lo_ptr = out_lo->data_ptr();
    }
    const size_t wsb = sdtw_cross_attention_workspace_bytes(&c.p);
    const Tensor ws = wsb > 0 ? workspace_of(wsb, q) : Tensor();
    const cudaStream_t stream = stream_of(q);
    check_status(sdtw_cross_attention(&c.p, out.data_ptr(), lo_ptr, lse_ptr, wsb > 0 ? ws.data_ptr() : nullptr, wsb, stream),
                 "cross_attention");
    maybe_sync_check(q, stream);
    return out;
}

Tensor cross_attention_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_x,
                            const OptTensor& lengths_y, int64_t bandwidth, double scale)
{
    return attention_forward(q, k, v, lengths_x, lengths_y, bandwidth, scale, false, nullptr, nullptr);
}

// Returns (out, out_lo, lse); out_lo is empty for float32.
std::tuple<Tensor, Tensor, Tensor> attention_cuda(const Tensor& q, const Tensor& k, const Tensor& v,
                                                  const OptTensor& lengths_x, const OptTensor& lengths_y,
                                                  int64_t bandwidth, double scale)
{
    Tensor out_lo, lse;
    const Tensor out = attention_forward(q, k, v, lengths_x, lengths_y, bandwidth, scale, true, &out_lo, &lse);
    return {out, out_lo, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward_cuda(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                           const Tensor& v, const Tensor& out, const Tensor& out_lo,
                                                           const Tensor& lse, const OptTensor& lengths_x,
                                                           const OptTensor& lengths_y, int64_t bandwidth, double scale)
{
    attention_checks(q, k, v, lengths_x, lengths_y, scale);
    const c10::cuda::CUDAGuard guard(q.device());
    AttentionCall c;
    fill_attention(c, q, k, v, lengths_x, lengths_y, bandwidth, scale, true);
    TORCH_CHECK(dout.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() && dout.device() == q.device(),
                "the gradient of the output must have the output's shape, dtype and device");
    TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == q.device() &&
                    out.is_contiguous(),
                "out is not the forward's");
    const bool lo = out_lo.numel() > 0;
    TORCH_CHECK(!lo || (out_lo.sizes() == q.sizes() && out_lo.scalar_type() == q.scalar_type() &&
                        out_lo.device() == q.device() && out_lo.is_contiguous()),
                "out_lo is not the forward's");
    TORCH_CHECK(lse.sizes() == at::IntArrayRef({c.p.B, c.p.Hq, c.p.N}) && lse.scalar_type() == at::kFloat &&
                    lse.device() == q.device() && lse.is_contiguous(),
                "lse is not the forward's");
    const Tensor g = tensor_core_rows(dout);
    const int64_t gs[3] = {g.stride(0), g.stride(1), g.stride(2)};
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                 dv = at::empty(v.sizes(), v.options());
    const size_t wsb = sdtw_cross_attention_backward_workspace_bytes(&c.p);
    const Tensor ws = wsb > 0 ? workspace_of(wsb, q) : Tensor();
    const cudaStream_t stream = stream_of(q);
    check_status(sdtw_cross_attention_backward(&c.p, out.data_ptr(), lo ? out_lo.data_ptr() : nullptr,
                                               lse.data_ptr<float>(), g.data_ptr(), gs, dq.data_ptr(), dk.data_ptr(),
                                               dv.data_ptr(), wsb > 0 ? ws.data_ptr() : nullptr, wsb, stream),
                 "cross_attention_backward");
    maybe_sync_check(q, stream);
    return {dq, dk, dv};
}

// ---------------------------------------------------------------------------------------------------
// Head norm with rotation
// ---------------------------------------------------------------------------------------------------
struct RotateCall {
    sdtw_rotate_problem p{};
    Tensor x, weight, lengths, positions;
};

void fill_rotate(RotateCall& c, const Tensor& x, const OptTensor& weight, const OptTensor& lengths,
                 const OptTensor& positions, int64_t rotary, double base, bool interleaved, double eps)
{
    TORCH_CHECK(x.dim() == 4, "x must be 4D (B, N, H, d)");
    const int64_t B = x.size(0), N = x.size(1), d = x.size(3);
    TORCH_CHECK(d >= 1 && d <= 256, "the head dimension must lie in [1, 256], got ", num(d));
    float_type(x, "x");
    cuda_tensor(x);
    TORCH_CHECK(rotary >= 0 && rotary <= d && rotary % 2 == 0,
                "rotary_dim must be even and lie in [0, d] = [0, ", num(d), "], got ", num(rotary));
    TORCH_CHECK(base > 0 && std::isfinite(base), "base must be positive");
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "eps must not be negative");
    lengths_check(lengths, B, x, "lengths");
    if (weight) {
        TORCH_CHECK(weight->dim() == 1 && weight->size(0) == d, "weight must have shape (", num(d), ",), got ", shape_of(*weight));
        TORCH_CHECK(weight->scalar_type() == x.scalar_type() || weight->scalar_type() == at::kFloat,
                    "weight must have x's dtype or float32");
        TORCH_CHECK(weight->device() == x.device(), "weight must be on ", x.device(), ", got ", weight->device());
        c.weight = weight->contiguous();
    }
    if (positions) {
        const auto st = positions->scalar_type();
        TORCH_CHECK(st == at::kFloat || st == at::kInt || st == at::kLong, "positions must be float32, int32 or int64");
        TORCH_CHECK(positions->sizes() == at::IntArrayRef({B, N}) || positions->sizes() == at::IntArrayRef({N}),
                    "positions must have shape (", num(B), ", ", num(N), ") or (", num(N), ",), got ", shape_of(*positions));
        TORCH_CHECK(positions->device() == x.device(), "positions must be on ", x.device(), ", got ",
                    positions->device());
        c.positions = *positions;
        c.p.positions = c.positions.data_ptr();
        c.p.position_kind = st == at::kFloat ? 0 : (st == at::kInt ? 1 : 2);
        const bool rows = positions->dim() == 2;
        c.p.position_stride[0] = rows ? c.positions.stride(0) : 0;
        c.p.position_stride[1] = c.positions.stride(rows ? 1 : 0);
    }
    if (lengths) c.lengths = lengths->contiguous();
    c.x = feature_rows(x);
    sdtw_rotate_problem& p = c.p;
    p.dtype = code_of(x.scalar_type());
    p.weight_f32 = c.weight.defined() && c.weight.scalar_type() == at::kFloat;
    p.x = c.x.data_ptr();
    for (int i = 0; i < 3; ++i) p.x_stride[i] = c.x.stride(i);
    p.B = B;
    p.N = N;
    p.H = x.size(2);
    p.d = d;
    p.weight = c.weight.defined() ? c.weight.data_ptr() : nullptr;
    p.lengths = c.lengths.defined() ? c.lengths.data_ptr() : nullptr;
    p.lengths_int32 = c.lengths.defined() && c.lengths.scalar_type() == at::kInt;
    p.rotary = rotary;
    p.interleaved = interleaved;
    p.base = base;
    p.eps = eps;
    p.err_word = error_word(x);
}

Tensor norm_rotate_cuda(const Tensor& x, const OptTensor& weight, const OptTensor& lengths,
                        const OptTensor& positions, int64_t rotary, double base, bool interleaved, double eps)
{
    cuda_tensor(x);
    const c10::cuda::CUDAGuard guard(x.device());
    RotateCall c;
    fill_rotate(c, x, weight, lengths, positions, rotary, base, interleaved, eps);
    const Tensor y = at::empty(x.sizes(), x.options());
    const cudaStream_t stream = stream_of(x);
    check_status(sdtw_norm_rotate(&c.p, y.data_ptr(), stream), "norm_rotate");
    maybe_sync_check(x, stream);
    return y;
}

// Returns (dx, dweight); dweight is empty when there is no weight or it is not asked for.
std::tuple<Tensor, Tensor> norm_rotate_backward_cuda(const Tensor& dy, const Tensor& x, const OptTensor& weight,
                                                     const OptTensor& lengths, const OptTensor& positions,
                                                     int64_t rotary, double base, bool interleaved, double eps,
                                                     bool need_weight)
{
    cuda_tensor(x);
    const c10::cuda::CUDAGuard guard(x.device());
    RotateCall c;
    fill_rotate(c, x, weight, lengths, positions, rotary, base, interleaved, eps);
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
                "the gradient of the output must have the output's shape, dtype and device");
    const Tensor g = feature_rows(dy);
    const int64_t gs[3] = {g.stride(0), g.stride(1), g.stride(2)};
    const bool dw = need_weight && weight.has_value();
    const Tensor dx = at::empty(x.sizes(), x.options());
    const Tensor dweight = dw ? at::empty({c.p.d}, weight->options()) : at::empty({0}, x.options());
    const size_t wsb = dw ? sdtw_norm_rotate_backward_workspace_bytes(c.p.d) : 0;
    const Tensor ws = dw ? workspace_of(wsb, x) : Tensor();
    const cudaStream_t stream = stream_of(x);
    check_status(sdtw_norm_rotate_backward(&c.p, g.data_ptr(), gs, dx.data_ptr(), dw ? dweight.data_ptr() : nullptr,
                                           dw ? ws.data_ptr() : nullptr, wsb, stream),
                 "norm_rotate_backward");
    maybe_sync_check(x, stream);
    return {dx, dweight};
}

// ---------------------------------------------------------------------------------------------------
// Global norm and clipping
// ---------------------------------------------------------------------------------------------------
int norm_kind_of(double norm_type)
{
    TORCH_CHECK(norm_type == 2.0 || (std::isinf(norm_type) && norm_type > 0), "norm_type must be 2 or inf, got ",
                num(norm_type));
    return norm_type == 2.0 ? SDTW_NORM_L2 : SDTW_NORM_MAX;
}

// The tensors as the kernels read them (dense memory, any order of dimensions) and whether one is float64.
bool tensor_checks(at::TensorList ts)
{
    bool wide = false;
    for (const Tensor& t : ts) {
        TORCH_CHECK(t.layout() == at::kStrided, "tensors must be dense, got a ", t.layout(), " tensor");
        const auto st = t.scalar_type();
        TORCH_CHECK(st == at::kFloat || st == at::kDouble || st == at::kHalf || st == at::kBFloat16,
                    "tensors must be float16, bfloat16, float32 or float64, got ", st);
        cuda_tensor(t);
        TORCH_CHECK(t.device() == ts[0].device(), "all tensors must be on one device, got ", ts[0].device(), " and ",
                    t.device());
        wide = wide || st == at::kDouble;
    }
    return wide;
}

bool is_dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

sdtw_tensor_ref ref_of(const Tensor& src, void* dst)
{
    return {src.data_ptr(), dst, src.numel(), static_cast<int32_t>(code_of(src.scalar_type())), 0};
}

// Where a tensor's entries lie: `width` bytes at every sum of a multiple of each stride (in bytes, largest first) below its size.
struct Places {
    struct Dim {
        int64_t size, stride;
    };
    std::vector<Dim> dims;
    int64_t width;
    int64_t extent(size_t from) const  // of the dimensions from `from` on
    {
        int64_t e = width;
        for (size_t i = from; i < dims.size(); ++i) e += (dims[i].size - 1) * dims[i].stride;
        return e;
    }
};

Places places_of(const Tensor& t)
{
    Places p;
    p.width = t.element_size();
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) > 0) p.dims.push_back({t.size(i), t.stride(i) * p.width});
    std::sort(p.dims.begin(), p.dims.end(), [](const Places::Dim& a, const Places::Dim& b) { return a.stride > b.stride; });
    while (!p.dims.empty() && p.dims.back().stride <= p.width) {  // neighbours without a gap are one piece
        p.width += (p.dims.back().size - 1) * p.dims.back().stride;
        p.dims.pop_back();
    }
    return p;
}

// Whether dimensions i.. of a and j.. of b, which begins `at` bytes behind a, share a byte. Extents that do not meet share none; rows of
// one pitch meet by their difference alone; otherwise the tensor with the longer pitch is taken row by row. After `steps` the
// answer is yes.
bool share(const Places& a, size_t i, const Places& b, size_t j, int64_t at, int& steps)
{
    if (at >= a.extent(i) || -at >= b.extent(j)) return false;
    const bool more_a = i < a.dims.size(), more_b = j < b.dims.size();
    if ((!more_a && !more_b) || --steps < 0) return true;
    const auto ceil = [](int64_t x, int64_t y) { return x / y + (x % y > 0); };
    const auto floor = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t pa = more_a ? a.dims[i].stride : 0, pb = more_b ? b.dims[j].stride : 0;
    const size_t ni = pa >= pb ? i + 1 : i, nj = pb >= pa ? j + 1 : j;
    const int64_t pitch = std::max(pa, pb), wa = a.extent(ni), wb = b.extent(nj);
    // x: a row of b less a row of a (one of them 0, where only one tensor has rows of this pitch).
    const int64_t first = std::max(pa >= pb ? 1 - a.dims[i].size : 0, ceil(1 - wb - at, pitch));
    const int64_t last = std::min(pb >= pa ? b.dims[j].size - 1 : 0, floor(wa - 1 - at, pitch));
    for (int64_t x = first; x <= last; ++x)
        if (share(a, ni, b, nj, at + x * pitch, steps)) return true;
    return false;
}

bool share_memory(const Tensor& a, const Tensor& b)
{
    int steps = 1 << 20;
    const int64_t at = static_cast<int64_t>(reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr()));
    return share(places_of(a), 0, places_of(b), 0, at, steps);
}

Tensor norm_result(const Tensor& like, bool wide)
{
    return at::empty({}, like.options().dtype(wide ? at::kDouble : at::kFloat));
}

Tensor global_norm_cuda(at::TensorList tensors, double norm_type)
{
    const int kind = norm_kind_of(norm_type);
    TORCH_CHECK(!tensors.empty(), "global_norm needs a tensor");
    const bool wide = tensor_checks(tensors);
    const c10::cuda::CUDAGuard guard(tensors[0].device());
    std::vector<Tensor> keep;
    std::vector<sdtw_tensor_ref> refs;
    refs.reserve(tensors.size());
    for (const Tensor& t : tensors) {
        if (!is_dense(t)) keep.push_back(t.contiguous());
        refs.push_back(ref_of(is_dense(t) ? t : keep.back(), nullptr));
    }
    const Tensor norm = norm_result(tensors[0], wide);
    const size_t wsb = sdtw_clip_workspace_bytes(static_cast<int64_t>(refs.size()));
    const Tensor ws = workspace_of(wsb, tensors[0]);
    check_status(sdtw_global_norm(refs.data(), static_cast<int64_t>(refs.size()), kind, norm.data_ptr(), wide,
                                  ws.data_ptr(), wsb, stream_of(tensors[0])),
                 "global_norm");
    return norm;
}

// out[i] = grads[i] * min(1, max_norm / (norm + 1e-6)); out may hold the gradients themselves. Returns the norm.
Tensor clip_grads_cuda(at::TensorList grads, at::TensorList out, double max_norm, double norm_type)
{
    const int kind = norm_kind_of(norm_type);
    TORCH_CHECK(max_norm >= 0, "max_norm must not be negative, got ", num(max_norm));
    TORCH_CHECK(!grads.empty(), "clip_grads needs a tensor");
    TORCH_CHECK(grads.size() == out.size(), "out must hold one tensor for each gradient, got ", num(out.size()), " for ",
                num(grads.size()));
    const bool wide = tensor_checks(grads);
    const c10::cuda::CUDAGuard guard(grads[0].device());
    struct Range {
        uintptr_t begin, end;
        size_t index;
        bool written;
        const Tensor* tensor;
    };
    std::vector<Range> ranges;
    std::vector<Tensor> keep;                          // copies of gradients that are not dense
    std::vector<std::pair<size_t, Tensor>> later;      // results that are copied to out[i] at the end
    std::vector<sdtw_tensor_ref> refs;
    ranges.reserve(2 * grads.size());
    refs.reserve(grads.size());
    const auto range_of = [](const Tensor& t, bool written, size_t i) {
        int64_t last = t.is_contiguous() ? t.numel() - 1 : 0;
        if (!t.is_contiguous())
            for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
        return Range{p, p + static_cast<uintptr_t>(last + 1) * t.element_size(), i, written, &t};
    };
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i], &o = out[i];
        TORCH_CHECK(o.sizes() == g.sizes() && o.scalar_type() == g.scalar_type() && o.device() == g.device() &&
                        o.layout() == at::kStrided,
                    "out[", num(i), "] must have the gradient's shape, dtype and device");
        TORCH_CHECK(g.numel() == 0 || is_dense(o) || at::has_internal_overlap(o) != at::MemOverlap::Yes, "out[", num(i),
                    "] holds several entries in one place");
        const bool alike = o.strides() == g.strides();
        if (g.numel() > 0) {
            ranges.push_back(range_of(o, true, i));
            if (!alike || o.data_ptr() != g.data_ptr()) ranges.push_back(range_of(g, false, i));
        }
        // Results that are not laid out as their gradient are scaled into a buffer that is, then copied.
        if (alike && is_dense(g)) {
            refs.push_back(ref_of(g, o.data_ptr()));
        } else {
            if (!is_dense(g)) keep.push_back(g.contiguous());
            const Tensor& src = is_dense(g) ? g : keep.back();
            if (is_dense(o) && o.strides() == src.strides()) {
                refs.push_back(ref_of(src, o.data_ptr()));
            } else {
                later.emplace_back(i, at::empty_like(src));
                refs.push_back(ref_of(src, later.back().second.data_ptr()));
            }
        }
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    std::vector<const Range*> open;  // those that end behind the present one's begin
    for (const Range& r : ranges) {
        size_t kept = 0;
        for (const Range* o : open) {
            if (o->end <= r.begin) continue;
            open[kept++] = o;
            TORCH_CHECK(!(o->written || r.written) || !share_memory(*o->tensor, *r.tensor), "clip_grads: tensor ", num(r.index),
                        " shares memory with another one that is written");
        }
        open.resize(kept);
        open.push_back(&r);
    }
    const Tensor norm = norm_result(grads[0], wide);
    const size_t wsb = sdtw_clip_workspace_bytes(static_cast<int64_t>(refs.size()));
    const Tensor ws = workspace_of(wsb, grads[0]);
    check_status(sdtw_clip_grads(refs.data(), static_cast<int64_t>(refs.size()), kind, max_norm, norm.data_ptr(), wide,
                                 ws.data_ptr(), wsb, stream_of(grads[0])),
                 "clip_grads");
    for (const auto& [i, t] : later)
        if (t.numel() > 0) out[i].copy_(t);
    for (const Tensor& o : out)
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return norm;
}

// ---------------------------------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename F>
auto typed_op(const char* name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
const auto& attention_op()
{
    static const auto op = typed_op<decltype(attention_cuda)>("torchsoftdtw_b200::attention");
    return op;
}
const auto& cross_attention_op()
{
    static const auto op = typed_op<decltype(cross_attention_cuda)>("torchsoftdtw_b200::cross_attention");
    return op;
}
const auto& attention_backward_op()
{
    static const auto op = typed_op<decltype(attention_backward_cuda)>("torchsoftdtw_b200::attention_backward");
    return op;
}
const auto& norm_rotate_op()
{
    static const auto op = typed_op<decltype(norm_rotate_cuda)>("torchsoftdtw_b200::norm_rotate");
    return op;
}
const auto& norm_rotate_backward_op()
{
    static const auto op = typed_op<decltype(norm_rotate_backward_cuda)>("torchsoftdtw_b200::norm_rotate_backward");
    return op;
}

OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor tensor_of(const OptTensor& t) { return t ? *t : Tensor(); }
// Whether a call belongs to a graph. Forward-mode tangents are refused rather than dropped.
bool wants_grad(const char* name, std::initializer_list<Tensor> ts)
{
    bool wants = false;
    for (const Tensor& t : ts) {
        if (!t.defined()) continue;
        TORCH_CHECK(!t._fw_grad(0).defined(), name, " has no forward-mode derivative");
        wants = wants || t.requires_grad();
    }
    return wants && at::GradMode::is_enabled();
}

// The gradients themselves are not differentiable: differentiating them raises.
variable_list twice(const char* name)
{
    TORCH_CHECK(false, name, " is differentiable once; its gradients have no gradient");
    return {};
}

struct AttentionBackward : torch::autograd::Function<AttentionBackward> {
    static variable_list forward(AutogradContext*, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& out, const Tensor& out_lo, const Tensor& lse, const OptTensor& lx,
                                 const OptTensor& ly, int64_t bandwidth, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [dq, dk, dv] = attention_backward_op().call(dout, q, k, v, out, out_lo, lse, lx, ly, bandwidth, scale);
        return {dq, dk, dv};
    }
    static variable_list backward(AutogradContext*, const variable_list&) { return twice("cross_attention"); }
};

std::tuple<Tensor, Tensor, Tensor> attention_backward_autograd(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                               const Tensor& v, const Tensor& out, const Tensor& out_lo,
                                                               const Tensor& lse, const OptTensor& lx, const OptTensor& ly,
                                                               int64_t bandwidth, double scale)
{
    if (wants_grad("cross_attention", {dout, q, k, v, out})) {
        const variable_list g = AttentionBackward::apply(dout, q, k, v, out, out_lo, lse, lx, ly, bandwidth, scale);
        return {g[0], g[1], g[2]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return attention_backward_op().call(dout, q, k, v, out, out_lo, lse, lx, ly, bandwidth, scale);
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lx,
                          const OptTensor& ly, int64_t bandwidth, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [out, out_lo, lse] = attention_op().call(q, k, v, lx, ly, bandwidth, scale);
        ctx->save_for_backward({q, k, v, out, out_lo, lse, tensor_of(lx), tensor_of(ly)});
        ctx->saved_data["bandwidth"] = bandwidth;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        const variable_list s = ctx->get_saved_variables();
        auto [dq, dk, dv] = attention_backward_op().call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], optional_of(s[6]),
                                                         optional_of(s[7]), ctx->saved_data["bandwidth"].toInt(),
                                                         ctx->saved_data["scale"].toDouble());
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor cross_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lx, const OptTensor& ly,
                                int64_t bandwidth, double scale)
{
    if (wants_grad("cross_attention", {q, k, v})) return CrossAttention::apply(q, k, v, lx, ly, bandwidth, scale);
    at::AutoDispatchBelowADInplaceOrView guard;
    return cross_attention_op().call(q, k, v, lx, ly, bandwidth, scale);
}

struct NormRotateBackward : torch::autograd::Function<NormRotateBackward> {
    static variable_list forward(AutogradContext*, const Tensor& dy, const Tensor& x, const OptTensor& weight,
                                 const OptTensor& lengths, const OptTensor& positions, int64_t rotary, double base,
                                 bool interleaved, double eps, bool need_weight)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [dx, dw] = norm_rotate_backward_op().call(dy, x, weight, lengths, positions, rotary, base, interleaved, eps,
                                                       need_weight);
        return {dx, dw};
    }
    static variable_list backward(AutogradContext*, const variable_list&) { return twice("norm_rotate"); }
};

std::tuple<Tensor, Tensor> norm_rotate_backward_autograd(const Tensor& dy, const Tensor& x, const OptTensor& weight,
                                                         const OptTensor& lengths, const OptTensor& positions,
                                                         int64_t rotary, double base, bool interleaved, double eps,
                                                         bool need_weight)
{
    if (wants_grad("norm_rotate", {dy, x, tensor_of(weight)})) {
        const variable_list g = NormRotateBackward::apply(dy, x, weight, lengths, positions, rotary, base, interleaved, eps,
                                                          need_weight);
        return {g[0], g[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return norm_rotate_backward_op().call(dy, x, weight, lengths, positions, rotary, base, interleaved, eps, need_weight);
}

struct NormRotate : torch::autograd::Function<NormRotate> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& lengths,
                          const OptTensor& positions, int64_t rotary, double base, bool interleaved, double eps)
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Tensor y = norm_rotate_op().call(x, weight, lengths, positions, rotary, base, interleaved, eps);
        ctx->save_for_backward({x, tensor_of(weight), tensor_of(lengths), tensor_of(positions)});
        ctx->saved_data["rotary"] = rotary;
        ctx->saved_data["base"] = base;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["need_weight"] = weight.has_value() && weight->requires_grad();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const bool need_weight = ctx->saved_data["need_weight"].toBool();
        auto [dx, dw] = norm_rotate_backward_op().call(
            grads[0], s[0], optional_of(s[1]), optional_of(s[2]), optional_of(s[3]), ctx->saved_data["rotary"].toInt(),
            ctx->saved_data["base"].toDouble(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["eps"].toDouble(),
            need_weight);
        return {dx, need_weight ? dw : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor norm_rotate_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& lengths, const OptTensor& positions,
                            int64_t rotary, double base, bool interleaved, double eps)
{
    if (wants_grad("norm_rotate", {x, tensor_of(weight)}))
        return NormRotate::apply(x, weight, lengths, positions, rotary, base, interleaved, eps);
    at::AutoDispatchBelowADInplaceOrView guard;
    return norm_rotate_op().call(x, weight, lengths, positions, rotary, base, interleaved, eps);
}

// CPU tensors: argument errors read like those of CUDA ones; then the device is refused.
Tensor cross_attention_cpu(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_x,
                           const OptTensor& lengths_y, int64_t bandwidth, double scale)
{
    (void)bandwidth;
    attention_checks(q, k, v, lengths_x, lengths_y, scale);
    return {};
}

std::tuple<Tensor, Tensor, Tensor> attention_cpu(const Tensor& q, const Tensor& k, const Tensor& v,
                                                 const OptTensor& lengths_x, const OptTensor& lengths_y,
                                                 int64_t bandwidth, double scale)
{
    cross_attention_cpu(q, k, v, lengths_x, lengths_y, bandwidth, scale);
    return {};
}

Tensor norm_rotate_cpu(const Tensor& x, const OptTensor& weight, const OptTensor& lengths, const OptTensor& positions,
                       int64_t rotary, double base, bool interleaved, double eps)
{
    RotateCall c;
    fill_rotate(c, x, weight, lengths, positions, rotary, base, interleaved, eps);
    return {};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torchsoftdtw_b200, m)
{
    m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths_x, Tensor? lengths_y, int bandwidth, float scale) "
          "-> Tensor");
    m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? lengths_x, Tensor? lengths_y, int bandwidth, float scale) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor out_lo, Tensor lse, "
          "Tensor? lengths_x, Tensor? lengths_y, int bandwidth, float scale) -> (Tensor, Tensor, Tensor)");
    m.def("norm_rotate(Tensor x, Tensor? weight, Tensor? lengths, Tensor? positions, int rotary_dim, float base, "
          "bool interleaved, float eps) -> Tensor");
    m.def("norm_rotate_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? lengths, Tensor? positions, "
          "int rotary_dim, float base, bool interleaved, float eps, bool need_weight) -> (Tensor, Tensor)");
    m.def("global_norm(Tensor[] tensors, float norm_type) -> Tensor");
    m.def("clip_grads(Tensor[] grads, Tensor(a!)[] out, float max_norm, float norm_type) -> Tensor");
}

TORCH_LIBRARY_IMPL(torchsoftdtw_b200, CUDA, m)
{
    m.impl("cross_attention", &cross_attention_cuda);
    m.impl("attention", &attention_cuda);
    m.impl("attention_backward", &attention_backward_cuda);
    m.impl("norm_rotate", &norm_rotate_cuda);
    m.impl("norm_rotate_backward", &norm_rotate_backward_cuda);
    m.impl("global_norm", &global_norm_cuda);
    m.impl("clip_grads", &clip_grads_cuda);
}

TORCH_LIBRARY_IMPL(torchsoftdtw_b200, CPU, m)
{
    m.impl("cross_attention", &cross_attention_cpu);
    m.impl("attention", &attention_cpu);
    m.impl("norm_rotate", &norm_rotate_cpu);
    m.impl("global_norm", &global_norm_cuda);
    m.impl("clip_grads", &clip_grads_cuda);
}

TORCH_LIBRARY_IMPL(torchsoftdtw_b200, Autograd, m)
{
    m.impl("cross_attention", &cross_attention_autograd);
    m.impl("attention_backward", &attention_backward_autograd);
    m.impl("norm_rotate", &norm_rotate_autograd);
    m.impl("norm_rotate_backward", &norm_rotate_backward_autograd);
    // Norms and clipped gradients are results, not steps of a graph.
    m.impl("global_norm", torch::CppFunction::makeFallthrough());
    m.impl("clip_grads", torch::CppFunction::makeFallthrough());
}
