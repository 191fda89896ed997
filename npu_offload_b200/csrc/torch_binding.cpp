// Torch-side half of the calls that allocate through torch (e4m3, routing in groups, balance loss, norm, adapters): checks, allocation of results and working memory, and
// the call of the C ABI.  These calls take a few microseconds on the GPU at one token; through Python and
// ctypes the host needed 11 us (quantiser, product) to 30 us (loss and gradient) for them.
//
// Refusals are ValueError, statuses of the library MoEError.  Results and working memory come from torch's
// allocator on the calling thread's current stream, which is also the one that the calls run on: working
// memory is a tensor here until its kernels are enqueued, and freed in the stream's order.
#include <torch/extension.h>

#include <ATen/EmptyTensor.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>

#include <string>

#include "../../include/moe_dp.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Plane {  // what a call needs of its data plane
    moe_ctx* ctx;
    at::Device device;
    int64_t H, F, E, K;
};

// Messages without streams: a host libstdc++ other than torch's may not share its locale facets.
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(const at::Device& d) {
    return std::string(d.is_cuda() ? "cuda" : "cpu") + (d.has_index() ? ":" + std::to_string((int)d.index()) : "");
}
template <class... A>
[[noreturn]] void refuse(const A&... parts) {
    throw py::value_error((text(parts) + ...));
}

void check(int status) {
    if (status != MOE_OK) py::module_::import("npu_offload_b200._lib").attr("check")(status);  // raises MoEError
}

std::string shape(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

std::string name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        case at::kBool: return "torch.bool";
        case at::kByte: return "torch.uint8";
        case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
        default: return "torch type " + std::to_string((int)t);
    }
}

// No call records an autograd graph: a gradient that one would drop in silence is refused.
void no_gradient(const char* name, const Tensor& t) {
    if (t.requires_grad() && at::GradMode::is_enabled())
        refuse(name, " requires a gradient, and this call records no autograd graph: pass it detached, or call under torch.no_grad()");
}

// A new tensor of the plane's device, straight from torch's allocator: at::empty takes 0.7 us on the host, this 0.4, and a call at
// one token has five.
Tensor fresh(const Plane& p, at::IntArrayRef sizes, at::ScalarType type) {
    if (!p.device.is_cuda()) return at::empty(sizes, at::TensorOptions(p.device).dtype(type));
    const c10::DeviceGuard guard(p.device);
    return at::detail::empty_generic(sizes, c10::GetAllocator(c10::DeviceType::CUDA), c10::DispatchKeySet(c10::DispatchKey::CUDA), type,
                                     c10::nullopt);
}

// t as a contiguous tensor of the plane's device, at a multiple of `align` bytes; other types and ranks are refused.
Tensor operand(const Plane& p, const char* name, Tensor t, std::initializer_list<at::ScalarType> types, int dims, int align = 1) {
    if (!t.defined() || t.device() != p.device) refuse(name, " must be a tensor on ", p.device);
    bool ok = false;
    for (at::ScalarType s : types) ok |= t.scalar_type() == s;
    if (!ok) refuse(name, " is ", name_of(t.scalar_type()), ", not ", name_of(*types.begin()));
    if (dims >= 0 && t.dim() != dims) refuse(name, " has ", t.dim(), " dimensions, not ", dims);
    no_gradient(name, t);
    if (!t.is_contiguous()) t = t.contiguous();
    if (align > 1 && (uintptr_t)t.data_ptr() % align) t = t.clone();
    return t;
}

struct Fp8 {
    Tensor q, scale;
};
Fp8 fp8(const Plane& p, const char* name, const Tensor& q, const Tensor& scale, int dims, int64_t block_rows) {
    const std::string qn = std::string(name) + ".q", sn = std::string(name) + ".scale";
    // Weights are read in place: a copy of them on every call would cost more than the call.
    if (block_rows > 1 && q.defined() && q.device() == p.device) {
        if (!q.is_contiguous()) refuse(qn, " must be contiguous");
        if ((uintptr_t)q.data_ptr() % 16) refuse(qn, " must be 16-byte aligned: clone it once");
    }
    Fp8 m{operand(p, qn.c_str(), q, {at::kFloat8_e4m3fn}, dims, 16), operand(p, sn.c_str(), scale, {at::kFloat}, dims)};
    const int64_t rows = m.q.size(-2), cols = m.q.size(-1);
    bool ok = m.scale.size(-2) == (rows + block_rows - 1) / block_rows && m.scale.size(-1) == (cols + 127) / 128;
    for (int i = 0; i < dims - 2; i++) ok &= m.scale.size(i) == m.q.size(i);
    if (!ok) refuse(sn, " is ", shape(m.scale.sizes()), " for values of ", shape(m.q.sizes()), " in blocks of ", block_rows, " x 128");
    return m;
}

Tensor output(const Plane& p, const c10::optional<Tensor>& out, at::IntArrayRef sizes, at::ScalarType type, bool bf16) {
    if (!out) {
        if (type != at::kFloat && !(bf16 && type == at::kBFloat16)) refuse("out_dtype ", name_of(type), " is neither torch.bfloat16 nor torch.float32");
        return fresh(p, sizes, type);
    }
    const at::ScalarType t = out->scalar_type();
    if (out->device() != p.device || (t != at::kFloat && !(bf16 && t == at::kBFloat16)) || out->sizes() != sizes || !out->is_contiguous() ||
        (uintptr_t)out->data_ptr() % 16)
        refuse("out must be a contiguous, 16-byte aligned ", shape(sizes), bf16 ? " bf16 or fp32" : " fp32", " tensor on ", p.device);
    no_gradient("out", *out);
    return *out;
}

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? MOE_DT_F32 : MOE_DT_BF16; }
Tensor workspace(const Plane& p, int64_t bytes) {  // negative: the call itself says what is out of range
    return bytes > 0 ? fresh(p, {bytes}, at::kByte) : Tensor();
}
template <class T>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
template <class T>
T* ptr(const c10::optional<Tensor>& t) {
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

std::pair<Tensor, Tensor> quantize_fp8(const Plane& p, Tensor x, int64_t block_rows, int64_t stream) {
    x = operand(p, "x", std::move(x), {at::kBFloat16, at::kFloat}, -1, 16);
    if (x.dim() < 2 || (block_rows != 1 && block_rows != 128))
        refuse("quantize_fp8 takes [..., rows, cols] and block_rows 1 or 128");
    const int64_t rows = x.size(-2), cols = x.size(-1);
    int64_t batch = 1;
    auto sizes = x.sizes().vec();
    for (int64_t i = 0; i + 2 < x.dim(); i++) batch *= sizes[i];
    sizes[sizes.size() - 2] = (rows + block_rows - 1) / block_rows;
    sizes[sizes.size() - 1] = (cols + 127) / 128;
    const Tensor q = fresh(p, x.sizes(), at::kFloat8_e4m3fn), scale = fresh(p, sizes, at::kFloat);
    check(moe_quantize_fp8(p.ctx, x.data_ptr(), dtype_of(x), batch, rows, cols, (int)block_rows, ptr<uint8_t>(q), ptr<float>(scale), 0,
                           (void*)stream));
    return {q, scale};
}

Tensor matmul_fp8(const Plane& p, const Tensor& xq, const Tensor& xs, const Tensor& wq, const Tensor& ws, at::ScalarType out_dtype,
                  const c10::optional<Tensor>& out, int64_t stream) {
    const Fp8 x = fp8(p, "x", xq, xs, 2, 1), w = fp8(p, "w", wq, ws, 2, 128);
    const int64_t M = x.q.size(0), K = x.q.size(1), N = w.q.size(0);
    if (w.q.size(1) != K) refuse("x has ", K, " columns, w ", w.q.size(1));
    const Tensor o = output(p, out, {M, N}, out_dtype, true);
    check(moe_matmul_fp8(p.ctx, M, N, K, ptr<uint8_t>(x.q), ptr<float>(x.scale), ptr<uint8_t>(w.q), ptr<float>(w.scale), o.data_ptr(),
                         dtype_of(o), 0, (void*)stream));
    return o;
}

Tensor experts_fp8(const Plane& p, Tensor x, const Tensor& gq, const Tensor& gs, const Tensor& dq, const Tensor& ds, Tensor idx, Tensor w,
                   at::ScalarType out_dtype, const c10::optional<Tensor>& out, bool accumulate, int64_t stream) {
    x = operand(p, "x", std::move(x), {at::kBFloat16}, 2, 16);
    const int64_t T = x.size(0);
    if (x.size(1) != p.H) refuse("x has ", x.size(1), " columns, the context ", p.H);
    const Fp8 gu = fp8(p, "gate_up", gq, gs, 4, 128), d = fp8(p, "down", dq, ds, 3, 128);
    const int64_t gshape[4] = {p.E, 2, p.F, p.H}, dshape[3] = {p.E, p.H, p.F}, pairs[2] = {T, p.K};
    if (gu.q.sizes() != at::IntArrayRef(gshape)) refuse("gate_up is ", shape(gu.q.sizes()), ", not ", shape(gshape));
    if (d.q.sizes() != at::IntArrayRef(dshape)) refuse("down is ", shape(d.q.sizes()), ", not ", shape(dshape));
    idx = operand(p, "idx", std::move(idx), {at::kInt}, 2);
    w = operand(p, "w", std::move(w), {at::kFloat}, 2);
    if (idx.sizes() != at::IntArrayRef(pairs) || w.sizes() != at::IntArrayRef(pairs))
        refuse("idx ", shape(idx.sizes()), " and w ", shape(w.sizes()), " must be ", shape(pairs));
    if (accumulate && !out) refuse("accumulate needs an out to add to");
    if (T > INT32_MAX) refuse("T=", T, " is out of range");
    const Tensor o = output(p, out, {T, p.H}, out_dtype, true);
    const int64_t n = moe_experts_fp8_workspace(p.ctx, (int)T);
    const Tensor ws = workspace(p, n);
    check(moe_experts_fp8(p.ctx, (int)T, ptr<uint16_t>(x), ptr<uint8_t>(gu.q), ptr<float>(gu.scale), ptr<uint8_t>(d.q), ptr<float>(d.scale),
                          ptr<int32_t>(idx), ptr<float>(w), o.data_ptr(), dtype_of(o), ptr<void>(ws), n,
                          accumulate ? MOE_F_ACCUMULATE : 0, (void*)stream));
    return o;
}

struct Sequences {
    Tensor logits;
    c10::optional<Tensor> offsets, mask;
    int64_t T, B;
};
Sequences sequences(const Plane& p, Tensor logits, c10::optional<Tensor> offsets, c10::optional<Tensor> mask) {
    if (logits.defined() && logits.requires_grad() && at::GradMode::is_enabled())
        refuse("balance_loss records no autograd graph: pass logits.detach() and use balance_loss_backward");
    logits = operand(p, "logits", std::move(logits), {at::kFloat}, 2);
    if (logits.size(1) != p.E) refuse("logits have ", logits.size(1), " columns, the context ", p.E, " experts");
    Sequences s{logits, {}, {}, logits.size(0), 1};
    if (offsets) {
        s.offsets = operand(p, "offsets", *offsets, {at::kInt}, 1);
        s.B = s.offsets->size(0) - 1;
        if (s.B < 1 || s.B > INT32_MAX) refuse("offsets need two entries at least");
    }
    if (mask) {
        s.mask = operand(p, "mask", *mask, {at::kBool, at::kByte}, 1);
        if (s.mask->size(0) != s.T) refuse("mask has ", s.mask->size(0), " tokens, logits ", s.T);
    }
    return s;
}

std::tuple<Tensor, Tensor, Tensor, c10::optional<Tensor>, c10::optional<Tensor>> balance_loss(const Plane& p, Tensor logits, Tensor idx,
                                                                                             c10::optional<Tensor> offsets,
                                                                                             c10::optional<Tensor> mask, int64_t stream) {
    const Sequences s = sequences(p, std::move(logits), std::move(offsets), std::move(mask));
    idx = operand(p, "idx", std::move(idx), {at::kInt}, 2);
    const int64_t pairs[2] = {s.T, p.K};
    if (idx.sizes() != at::IntArrayRef(pairs)) refuse("idx is ", shape(idx.sizes()), ", not ", shape(pairs));
    const Tensor loss = fresh(p, {}, at::kFloat), counts = fresh(p, {s.B, p.E}, at::kInt), tokens = fresh(p, {s.B + 1}, at::kInt);
    const int64_t n = moe_balance_loss_workspace(p.ctx, s.T, (int)s.B);
    const Tensor ws = workspace(p, n);
    check(moe_balance_loss(p.ctx, s.T, ptr<float>(s.logits), ptr<int32_t>(idx), ptr<int32_t>(s.offsets), (int)s.B, ptr<uint8_t>(s.mask),
                           ptr<float>(loss), ptr<int32_t>(counts), ptr<int32_t>(tokens), ptr<void>(ws), n, 0, (void*)stream));
    return {loss, counts, tokens, s.offsets, s.mask};
}

Tensor balance_loss_backward(const Plane& p, Tensor logits, Tensor counts, Tensor tokens, c10::optional<Tensor> offsets,
                             c10::optional<Tensor> mask, c10::optional<Tensor> grad, const c10::optional<Tensor>& out, int64_t stream) {
    const Sequences s = sequences(p, std::move(logits), std::move(offsets), std::move(mask));
    counts = operand(p, "stats.counts", std::move(counts), {at::kInt}, 2);
    tokens = operand(p, "stats.tokens", std::move(tokens), {at::kInt}, 1);
    if (counts.size(0) != s.B || counts.size(1) != p.E || tokens.size(0) != s.B + 1) refuse("stats are of other sequences");
    if (grad) grad = operand(p, "grad", *grad, {at::kFloat}, 0);
    const Tensor o = output(p, out, {s.T, p.E}, at::kFloat, false);
    check(moe_balance_loss_backward(p.ctx, s.T, ptr<float>(s.logits), ptr<int32_t>(s.offsets), (int)s.B, ptr<uint8_t>(s.mask),
                                    ptr<int32_t>(counts), ptr<int32_t>(tokens), ptr<float>(grad), ptr<float>(o), 0, (void*)stream));
    return o;
}

struct Rows {  // [..., C] as T rows
    int64_t T, C;
};
Rows rows_of(const char* name, const Tensor& t) {
    if (t.dim() < 1 || t.size(-1) < 1) refuse(name, " must be [..., C] with a column at least, not ", shape(t.sizes()));
    return {t.numel() / t.size(-1), t.size(-1)};
}
Tensor norm_weight(const Plane& p, Tensor w, int64_t C) {
    w = operand(p, "weight", std::move(w), {at::kBFloat16, at::kFloat}, 1, 16);
    if (w.size(0) != C) refuse("weight has ", w.size(0), " values, the rows ", C);
    return w;
}

std::tuple<c10::optional<Tensor>, c10::optional<Tensor>, c10::optional<Tensor>, Tensor, Tensor> add_norm(
    const Plane& p, Tensor x, Tensor weight, c10::optional<Tensor> residual, double eps, c10::optional<at::ScalarType> out_dtype, bool fp8,
    int64_t stream) {
    x = operand(p, "x", std::move(x), {at::kBFloat16, at::kFloat}, -1, 16);
    const Rows n = rows_of("x", x);
    weight = norm_weight(p, std::move(weight), n.C);
    if (residual) {
        residual = operand(p, "residual", *residual, {at::kBFloat16, at::kFloat}, -1, 16);
        if (residual->sizes() != x.sizes()) refuse("residual is ", shape(residual->sizes()), ", x ", shape(x.sizes()));
    }
    if (out_dtype && *out_dtype != at::kBFloat16 && *out_dtype != at::kFloat)
        refuse("out_dtype ", name_of(*out_dtype), " is neither torch.bfloat16 nor torch.float32");
    if (!out_dtype && !fp8) refuse("neither an out_dtype nor fp8 is wanted");
    if (fp8 && n.C % 16) refuse("fp8 rows are a multiple of 16, not ", n.C, " columns");
    c10::optional<Tensor> y, q, scale;
    if (out_dtype) y = fresh(p, x.sizes(), *out_dtype);
    if (fp8) {
        auto sizes = x.sizes().vec();
        sizes.back() = (n.C + 127) / 128;
        q = fresh(p, x.sizes(), at::kFloat8_e4m3fn);
        scale = fresh(p, sizes, at::kFloat);
    }
    const Tensor sum = residual ? fresh(p, x.sizes(), residual->scalar_type()) : x;
    const Tensor rstd = fresh(p, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    check(moe_add_norm(p.ctx, n.T, n.C, x.data_ptr(), dtype_of(x), ptr<void>(residual), dtype_of(sum), weight.data_ptr(), dtype_of(weight),
                       (float)eps, residual ? sum.data_ptr() : nullptr, ptr<void>(y), y ? dtype_of(*y) : MOE_DT_BF16, ptr<uint8_t>(q),
                       ptr<float>(scale), ptr<float>(rstd), 0, (void*)stream));
    return {y, q, scale, sum, rstd};
}

std::pair<Tensor, c10::optional<Tensor>> add_norm_backward(const Plane& p, Tensor dy, Tensor sum, Tensor weight, Tensor rstd,
                                                          c10::optional<Tensor> dsum, bool weight_grad, int64_t stream) {
    dy = operand(p, "dy", std::move(dy), {at::kBFloat16, at::kFloat}, -1, 16);
    sum = operand(p, "sum", std::move(sum), {at::kBFloat16, at::kFloat}, -1, 16);
    const Rows n = rows_of("sum", sum);
    weight = norm_weight(p, std::move(weight), n.C);
    rstd = operand(p, "rstd", std::move(rstd), {at::kFloat}, (int)sum.dim() - 1);
    if (dy.sizes() != sum.sizes()) refuse("dy is ", shape(dy.sizes()), ", sum ", shape(sum.sizes()));
    if (rstd.sizes() != sum.sizes().slice(0, sum.dim() - 1)) refuse("rstd is ", shape(rstd.sizes()), " for a sum of ", shape(sum.sizes()));
    if (dsum) {
        dsum = operand(p, "dsum", *dsum, {sum.scalar_type()}, -1, 16);
        if (dsum->sizes() != sum.sizes()) refuse("dsum is ", shape(dsum->sizes()), ", sum ", shape(sum.sizes()));
    }
    const Tensor dx = fresh(p, sum.sizes(), sum.scalar_type());
    c10::optional<Tensor> dw;
    int64_t bytes = 0;
    if (weight_grad) {
        dw = fresh(p, {n.C}, at::kFloat);
        bytes = moe_add_norm_backward_workspace(p.ctx, n.T, n.C);
    }
    const Tensor ws = workspace(p, bytes);
    check(moe_add_norm_backward(p.ctx, n.T, n.C, dy.data_ptr(), dtype_of(dy), sum.data_ptr(), dtype_of(sum), ptr<void>(dsum),
                                weight.data_ptr(), dtype_of(weight), ptr<float>(rstd), dx.data_ptr(), ptr<float>(dw), ptr<void>(ws), bytes,
                                0, (void*)stream));
    return {dx, dw};
}

Tensor router_logits(const Plane& p, Tensor t) {
    t = operand(p, "logits", std::move(t), {at::kFloat}, 2);
    if (t.size(1) != p.E) refuse("logits are ", shape(t.sizes()), ", the context has ", p.E, " experts");
    return t;
}

std::pair<Tensor, Tensor> route_groups(const Plane& p, Tensor logits, int64_t groups, int64_t top_groups, c10::optional<Tensor> bias,
                                       bool renormalize, double scale, int64_t stream) {
    logits = router_logits(p, std::move(logits));
    if (bias) {
        bias = operand(p, "bias", bias->detach(), {at::kFloat}, 1);  // (it only selects: no gradient is lost)
        if (bias->size(0) != p.E) refuse("bias is ", shape(bias->sizes()), ", the context has ", p.E, " experts");
    }
    if (groups < INT32_MIN || groups > INT32_MAX || top_groups < INT32_MIN || top_groups > INT32_MAX) refuse("groups are out of range");
    const int64_t T = logits.size(0);
    const Tensor idx = fresh(p, {T, p.K}, at::kInt), w = fresh(p, {T, p.K}, at::kFloat);
    check(moe_route_groups(p.ctx, T, ptr<float>(logits), ptr<float>(bias), (int)groups, (int)top_groups, renormalize, (float)scale,
                           ptr<int32_t>(idx), ptr<float>(w), 0, (void*)stream));
    return {idx, w};
}

Tensor route_backward(const Plane& p, Tensor logits, Tensor idx, Tensor dw, bool renormalize, double scale, const c10::optional<Tensor>& out,
                      bool accumulate, int64_t stream) {
    logits = router_logits(p, std::move(logits));
    const int64_t T = logits.size(0), pairs[2] = {T, p.K};
    idx = operand(p, "idx", std::move(idx), {at::kInt}, 2);
    dw = operand(p, "dw", std::move(dw), {at::kFloat}, 2);
    if (idx.sizes() != at::IntArrayRef(pairs) || dw.sizes() != at::IntArrayRef(pairs))
        refuse("idx ", shape(idx.sizes()), " and dw ", shape(dw.sizes()), " must be ", shape(pairs));
    if (accumulate && !out) refuse("accumulate needs an out to add to");
    const Tensor o = output(p, out, {T, p.E}, at::kFloat, false);
    check(moe_route_backward(p.ctx, T, ptr<float>(logits), ptr<int32_t>(idx), ptr<float>(dw), renormalize, (float)scale, ptr<float>(o),
                             accumulate ? MOE_F_ACCUMULATE : 0, (void*)stream));
    return o;
}

// Read in place, like the e4m3 weights: never copied.
Tensor adapter(const Plane& p, const char* name, const Tensor& t) {
    if (t.defined() && t.device() == p.device) {
        if (!t.is_contiguous()) refuse(name, " must be contiguous");
        if ((uintptr_t)t.data_ptr() % 16) refuse(name, " must be 16-byte aligned: clone it once");
    }
    return operand(p, name, t, {at::kBFloat16}, 3, 16);
}

Tensor add_lora(const Plane& p, Tensor base, Tensor x, const Tensor& at_a, const Tensor& at_b, Tensor ids, c10::optional<Tensor> scale,
                const c10::optional<Tensor>& out, int64_t stream) {
    base = operand(p, "base", std::move(base), {at::kBFloat16, at::kFloat}, 2, 16);
    x = operand(p, "x", std::move(x), {at::kBFloat16}, 2, 16);
    const Tensor a = adapter(p, "a", at_a), b = adapter(p, "b", at_b);
    const int64_t T = x.size(0), K = x.size(1), N = b.size(1), r = a.size(1), n = a.size(0);
    if (a.size(2) != K) refuse("a is ", shape(a.sizes()), " for x of ", K, " columns");
    if (b.size(0) != n || b.size(2) != r) refuse("b is ", shape(b.sizes()), " beside a of ", shape(a.sizes()));
    if (base.size(0) != T || base.size(1) != N) refuse("base is ", shape(base.sizes()), ", not (", T, ", ", N, ")");
    ids = operand(p, "ids", std::move(ids), {at::kInt}, 1);
    if (ids.size(0) != T) refuse("ids has ", ids.size(0), " tokens, x ", T);
    if (scale) {
        scale = operand(p, "scale", *scale, {at::kFloat}, 1);
        if (scale->size(0) != n) refuse("scale has ", scale->size(0), " values for ", n, " adapters");
    }
    const Tensor o = output(p, out, {T, N}, base.scalar_type(), true);
    if (o.scalar_type() != base.scalar_type()) refuse("out is ", name_of(o.scalar_type()), ", base ", name_of(base.scalar_type()));
    const int64_t bytes = moe_add_lora_workspace(p.ctx, T, r, n);
    const Tensor ws = workspace(p, bytes);
    check(moe_add_lora(p.ctx, T, K, N, r, n, base.data_ptr(), ptr<uint16_t>(x), ptr<uint16_t>(a), ptr<uint16_t>(b), ptr<int32_t>(ids),
                       ptr<float>(scale), o.data_ptr(), dtype_of(o), ptr<void>(ws), bytes, 0, (void*)stream));
    return o;
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
    m.doc() = "Checks, allocation and calls of the entry points of libmoe_dp.so that allocate through torch.";
    py::class_<Plane>(m, "Plane").def(py::init([](int64_t ctx, at::Device device, int64_t H, int64_t F, int64_t E, int64_t K) {
        return Plane{(moe_ctx*)ctx, device, H, F, E, K};
    }));
    m.def("quantize_fp8", &quantize_fp8);
    m.def("matmul_fp8", &matmul_fp8);
    m.def("experts_fp8", &experts_fp8);
    m.def("balance_loss", &balance_loss);
    m.def("balance_loss_backward", &balance_loss_backward);
    m.def("route_groups", &route_groups);
    m.def("route_backward", &route_backward);
    m.def("add_lora", &add_lora);
    m.def("add_norm", &add_norm);
    m.def("add_norm_backward", &add_norm_backward);
}
