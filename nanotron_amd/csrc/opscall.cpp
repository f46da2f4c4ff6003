// Host side of the operators of ntops.h: checks of tensors, allocation, autograd, and the C-ABI calls.
//
// A call of a small operator is host time (a norm of one token: 3 us of GPU), so the path from Python to the launch is one
// native call, and autograd's nodes are C++ as well: backward runs on autograd's device thread without Python.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ntops.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

void call(int rc, const char* what) { TORCH_CHECK(rc == NTFP8_OK, what, " failed: ", ntfp8_strerror(rc), " (code ", rc, ")"); }
void* stream_of(const Tensor& t) { return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream()); }
void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int code_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return NTFP8_F32;
        case at::kHalf: return NTFP8_F16;
        case at::kBFloat16: return NTFP8_BF16;
        default: TORCH_CHECK_TYPE(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}
void on_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be on a CUDA device (there is no CPU implementation), got ", t.device());
    TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " must be a dense tensor");
}
void same_device(const Tensor& t, const Tensor& x, const char* name) {
    on_gpu(t, name);
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
}

// The operators here are differentiable once, and in reverse: what asks for more is told so instead of given zeros
void once(const char* name) { TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once: its backward pass cannot be recorded (create_graph)"); }
void no_tangent(const Tensor& t, const char* name) { TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name, " has no forward-mode derivative"); }

// x as rows of its last dimension that a kernel can walk with one stride
struct Rows {
    Tensor t;
    int64_t rows, cols, stride;
};
Rows rows_of(const Tensor& x) {
    const int64_t cols = x.size(-1);
    Rows r{x, cols ? x.numel() / cols : 0, cols, cols};
    if (x.is_contiguous()) return r;
    if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= cols) {
        r.stride = x.size(0) > 1 ? x.stride(0) : cols;
        return r;
    }
    r.t = x.contiguous();
    return r;
}

// row `i` of a dense 2-D tensor
Tensor row_of(const Tensor& t, int64_t i) {
    Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(t.storage()), t.key_set(), t.dtype());
    const int64_t size = t.size(1), stride = 1;
    v.unsafeGetTensorImpl()->set_sizes_and_strides(size, stride, t.storage_offset() + i * size);
    return v;
}

// ---------------------------------------------------------------------------------------------- layer norm
struct Norm {
    Tensor y, stats;   // stats: the rows' means and, behind them, their 1 / root of the variance
    Rows x;
};
Norm norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool keep) {
    Norm n{Tensor(), Tensor(), rows_of(x)};
    n.y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (keep) n.stats = at::empty({2, n.x.rows}, x.options().dtype(at::kFloat));
    if (x.numel() == 0) return n;
    const Tensor wd = w.defined() ? w.contiguous() : w, bd = b.defined() ? b.contiguous() : b;
    const int xd = code_of(x, "x"), wc = w.defined() ? code_of(w, "weight") : b.defined() ? code_of(b, "bias") : xd;
    float* const mean = static_cast<float*>(at_or_null(n.stats));
    call(ntops_layer_norm_forward(n.x.t.data_ptr(), xd, n.x.rows, n.x.cols, n.x.stride, at_or_null(wd), at_or_null(bd), wc, (float)eps, n.y.data_ptr(),
                                  mean, mean ? mean + n.x.rows : nullptr, stream_of(x)),
         "ntops_layer_norm_forward");
    return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    // gx, gw, gb: which gradients are wanted
    static Variable forward(AutogradContext* ctx, const Variable& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps, bool gx, bool gw, bool gb) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        Guard guard(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->saved_data["want"] = (int64_t)(gx | gw << 1 | gb << 2);
        Norm n = norm_forward(x, w, b, eps, true);
        // (a non-dense x is saved as the dense rows that were made of it: one copy serves both passes)
        ctx->save_for_backward({n.x.t.is_same(x) ? x : n.x.t, w, b, n.stats});
        return n.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("layer_norm");
        const variable_list s = ctx->get_saved_variables();
        const Variable &x = s[0], &w = s[1], &b = s[2];
        Guard guard(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t want = ctx->saved_data["want"].toInt();
        const bool gx = want & 1, gw = want & 2, gb = want & 4;
        if (!grads[0].defined()) return variable_list(7);
        Tensor dx, dw, db;
        const auto given = [&] { return variable_list{dx, dw, db, Variable(), Variable(), Variable(), Variable()}; };
        if (gx) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
        if (x.numel() == 0) {
            if (gw) dw = at::zeros_like(w);
            if (gb) db = at::zeros_like(b);
            return given();
        }
        const Rows xr = rows_of(x), gr = rows_of(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()));
        const int xd = code_of(x, "x"), wc = w.defined() ? code_of(w, "weight") : b.defined() ? code_of(b, "bias") : xd;
        if (gw && gb) {   // (one type: one allocation, and two views of it without a dispatch each)
            const Tensor both = at::empty({2, xr.cols}, w.options().memory_format(at::MemoryFormat::Contiguous));
            dw = row_of(both, 0);
            db = row_of(both, 1);
        } else if (gw) {
            dw = at::empty(w.sizes(), w.options().memory_format(at::MemoryFormat::Contiguous));
        } else if (gb) {
            db = at::empty(b.sizes(), b.options().memory_format(at::MemoryFormat::Contiguous));
        }
        Tensor scratch;
        if (gw || gb) scratch = at::empty({ntops_layer_norm_scratch(xd, xr.rows, xr.cols)}, x.options().dtype(at::kByte));
        const Tensor wd = w.defined() ? w.contiguous() : w;
        call(ntops_layer_norm_backward(gr.t.data_ptr(), gr.stride, xr.t.data_ptr(), xd, xr.rows, xr.cols, xr.stride, at_or_null(wd), wc, s[3].const_data_ptr<float>(),
                                       s[3].const_data_ptr<float>() + xr.rows, at_or_null(dx), at_or_null(dw), at_or_null(db), at_or_null(scratch), stream_of(x)),
             "ntops_layer_norm_backward");
        return given();
    }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    on_gpu(x, "x");
    code_of(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have a last dimension to normalise over, got shape ", x.sizes());
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(w, "weight"), std::pair<const Tensor&, const char*>(b, "bias")}) {
        if (!t.defined()) continue;
        same_device(t, x, name);
        code_of(t, name);
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1), name, " must have shape [", x.size(-1), "], got ", t.sizes());
        TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), name, " must be float32 or of the type of x (", x.scalar_type(), "), got ",
                         t.scalar_type());
    }
    TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias must have one type");
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
    for (const Tensor* t : {&x, &w, &b}) no_tangent(*t, "layer_norm");
    const bool gx = x.requires_grad(), gw = w.defined() && w.requires_grad(), gb = b.defined() && b.requires_grad();
    if (at::GradMode::is_enabled() && (gx || gw || gb)) return LayerNorm::apply(x, weight, bias, eps, gx, gw, gb);
    Guard guard(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    return norm_forward(x, w, b, eps, false).y;
}

// ---------------------------------------------------------------------------------------------- norms around a block
bool floats(const Tensor& t, const Tensor& x) { return t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(); }
Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }

struct Norms {
    Rows x, residual, gate;
    Tensor w, pw, y, h, stats;   // stats: 1 / rms of the rows of x and, behind them, of h
};
// what both passes hand to the library
ntops_rms_norm_desc norms_desc(const Norms& n, const Tensor& x, const Tensor& residual, const Tensor& gate, double eps, double scale) {
    ntops_rms_norm_desc d = {};
    d.x = n.x.t.data_ptr(), d.rows = n.x.rows, d.cols = n.x.cols, d.x_stride = n.x.stride;
    d.x_dtype = code_of(x, "x"), d.residual_dtype = residual.defined() ? code_of(residual, "residual") : d.x_dtype;
    d.gate_kind = !gate.defined() ? NTOPS_GATE_NONE : gate.dim() == 1 ? NTOPS_GATE_CHANNEL : NTOPS_GATE_ELEMENT;
    d.gate = at_or_null(n.gate.t), d.gate_stride = n.gate.stride;
    d.weight = at_or_null(n.w), d.post_weight = at_or_null(n.pw);
    const Tensor& one = n.w.defined() ? n.w : n.pw.defined() ? n.pw : n.gate.t;
    d.w_dtype = n.w.defined() || n.pw.defined() || d.gate_kind == NTOPS_GATE_CHANNEL ? code_of(one, "weight") : d.x_dtype;
    d.eps = (float)eps, d.residual_scale = (float)scale;
    if (n.stats.defined()) {
        d.second = n.stats.data_ptr<float>() + n.x.rows;
        if (n.pw.defined()) d.first = n.stats.data_ptr<float>();
    }
    return d;
}
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Norms norms_of(const Tensor& x, const Tensor& gate, const Tensor& w, const Tensor& pw) {
    Norms n;
    n.x = rows_of(x);
    n.w = contiguous(w), n.pw = contiguous(pw);
    if (gate.defined()) n.gate = gate.dim() == 1 ? Rows{gate.contiguous(), 1, gate.size(0), gate.size(0)} : rows_of(gate);
    return n;
}
Norms norms_forward(const Tensor& x, const Tensor& residual, const Tensor& w, const Tensor& pw, const Tensor& gate, double eps, double scale, bool keep) {
    Norms n = norms_of(x, gate, w, pw);
    n.y = dense_like(x);
    if (residual.defined()) n.h = dense_like(residual);
    if (keep) n.stats = at::empty({2, n.x.rows}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    if (x.numel() == 0) return n;
    ntops_rms_norm_desc d = norms_desc(n, x, residual, gate, eps, scale);
    if (residual.defined()) {
        n.residual = rows_of(residual);
        d.residual = n.residual.t.data_ptr(), d.residual_stride = n.residual.stride, d.h = n.h.data_ptr();
    }
    d.y = n.y.data_ptr();
    call(ntops_rms_norm_forward(&d, stream_of(x)), "ntops_rms_norm_forward");
    return n;
}

enum { kWantX = 1, kWantResidual = 2, kWantWeight = 4, kWantPost = 8, kWantGate = 16 };
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    // outputs: y, and h where there is a residual
    static variable_list forward(AutogradContext* ctx, const Variable& x, const std::optional<Tensor>& residual_, const std::optional<Tensor>& weight, const std::optional<Tensor>& post,
                                 const std::optional<Tensor>& gate_, double eps, double scale, int64_t want) {
        const Tensor residual = residual_.value_or(Tensor()), w = weight.value_or(Tensor()), pw = post.value_or(Tensor()), gate = gate_.value_or(Tensor());
        Guard guard(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Norms n = norms_forward(x, residual, w, pw, gate, eps, scale, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["want"] = want;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["scale"] = scale;
        // x itself is read again where a norm or a gate stands behind it, or where it is what the one norm reads
        const bool again = !residual.defined() || pw.defined() || gate.defined();
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->save_for_backward({again ? (n.x.t.is_same(x) ? x : n.x.t) : Tensor(), n.h, w, pw, gate, n.stats});
        if (!residual.defined()) return {n.y};
        return {n.y, n.h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("rms_norm");
        const variable_list s = ctx->get_saved_variables();
        const Variable &x_ = s[0], &h = s[1], &w = s[2], &pw = s[3], &gate = s[4];
        const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        const int64_t want = ctx->saved_data["want"].toInt();
        if (!dy.defined() && !dh.defined()) return variable_list(8);
        const Tensor& some = dy.defined() ? dy : dh;
        Guard guard(some.device());
        at::AutoDispatchBelowADInplaceOrView below;
        // the type of x is that of y; where x is not kept (a residual, no norm and no gate) its shape is that of h
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const auto xo = some.options().dtype(type).memory_format(at::MemoryFormat::Contiguous);
        const bool residual = h.defined();
        const double scale = ctx->saved_data["scale"].toDouble();
        Tensor dx, dr, dw, dpw, dgate;
        // one gradient serves both where they are equal
        const bool same = residual && !pw.defined() && !gate.defined() && scale == 1.0 && h.scalar_type() == type;
        if ((want & kWantX) || (same && (want & kWantResidual))) dx = at::empty(shape, xo);
        if ((want & kWantResidual) && !same) dr = dense_like(h);
        if (want & kWantWeight) dw = dense_like(w);
        if (want & kWantPost) dpw = dense_like(pw);
        if (want & kWantGate) dgate = dense_like(gate);
        const auto given = [&] { return variable_list{want & kWantX ? dx : Tensor(), same && (want & kWantResidual) ? dx : dr, dw, dpw, dgate, Tensor(), Tensor(), Tensor()}; };
        if (c10::multiply_integers(shape) == 0) {
            for (Tensor* t : {&dw, &dpw, &dgate})
                if (t->defined()) t->zero_();
            return given();
        }
        const Tensor x = x_.defined() ? x_ : h;   // (not read where it was not kept)
        Norms n = norms_of(x, gate, w, pw);
        n.stats = s[5];
        ntops_rms_norm_desc d = norms_desc(n, x, h, gate, ctx->saved_data["eps"].toDouble(), scale);
        d.x_dtype = type == at::kFloat ? NTFP8_F32 : type == at::kHalf ? NTFP8_F16 : NTFP8_BF16;
        if (!w.defined() && !pw.defined() && d.gate_kind != NTOPS_GATE_CHANNEL) d.w_dtype = d.x_dtype;
        d.h = at_or_null(h);
        ntops_rms_norm_grads g = {};
        Rows gy, gh;
        if (dy.defined()) {
            gy = rows_of(dy.scalar_type() == type ? dy : dy.to(type));
            g.dy = gy.t.data_ptr(), g.dy_stride = gy.stride;
        }
        if (dh.defined()) {
            gh = rows_of(dh.scalar_type() == h.scalar_type() ? dh : dh.to(h.scalar_type()));
            g.dh = gh.t.data_ptr(), g.dh_stride = gh.stride;
        }
        g.dx = at_or_null(dx), g.dresidual = at_or_null(dr), g.dgate = at_or_null(dgate), g.dweight = at_or_null(dw), g.dpost_weight = at_or_null(dpw);
        Tensor scratch;
        if (dw.defined() || dpw.defined() || (dgate.defined() && d.gate_kind == NTOPS_GATE_CHANNEL)) {
            scratch = at::empty({ntops_rms_norm_scratch(&d)}, some.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
            g.scratch = scratch.data_ptr();
        }
        call(ntops_rms_norm_backward(&d, &g, stream_of(some)), "ntops_rms_norm_backward");
        return given();
    }
};

// y, and h where there is a residual
std::vector<Tensor> rms_norm(const Tensor& x, const std::optional<Tensor>& residual_, const std::optional<Tensor>& weight, const std::optional<Tensor>& post, const std::optional<Tensor>& gate_,
                             double eps, double scale) {
    const Tensor residual = residual_.value_or(Tensor()), w = weight.value_or(Tensor()), pw = post.value_or(Tensor()), gate = gate_.value_or(Tensor());
    on_gpu(x, "x");
    code_of(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have a last dimension to normalise over, got shape ", x.sizes());
    const int64_t cols = x.size(-1), most = x.scalar_type() == at::kFloat ? 8192 : 16384;
    TORCH_CHECK_VALUE(cols <= most, "x may have ", most, " columns at most as ", x.scalar_type(), ", got ", cols);
    if (residual.defined()) {
        same_device(residual, x, "residual");
        code_of(residual, "residual");
        TORCH_CHECK_VALUE(residual.sizes() == x.sizes(), "residual must have the shape of x, ", x.sizes(), ", got ", residual.sizes());
        TORCH_CHECK_TYPE(floats(residual, x), "residual must be float32 or of the type of x (", x.scalar_type(), "), got ", residual.scalar_type());
    }
    Tensor first;   // the vectors have one type
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(w, "weight"), std::pair<const Tensor&, const char*>(pw, "post_weight"), std::pair<const Tensor&, const char*>(gate, "gate")}) {
        if (!t.defined()) continue;
        same_device(t, x, name);
        code_of(t, name);
        if (&t == &gate && t.dim() != 1) {
            TORCH_CHECK_VALUE(t.sizes() == x.sizes(), "gate must have shape [", cols, "] or that of x, ", x.sizes(), ", got ", t.sizes());
            TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), "a gate for every element must be of the type of x (", x.scalar_type(), "), got ", t.scalar_type());
            continue;
        }
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == cols, name, " must have shape [", cols, "], got ", t.sizes());
        TORCH_CHECK_TYPE(floats(t, x), name, " must be float32 or of the type of x (", x.scalar_type(), "), got ", t.scalar_type());
        TORCH_CHECK_TYPE(!first.defined() || first.scalar_type() == t.scalar_type(), "weight, post_weight and a channel's gate must have one type");
        first = t;
    }
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
    TORCH_CHECK_VALUE(std::isfinite(scale), "residual_scale must be finite");
    for (const Tensor* t : {&x, &residual, &w, &pw, &gate}) no_tangent(*t, "rms_norm");
    int64_t want = 0;
    const auto wants = [&](const Tensor& t, int64_t bit) { want |= t.defined() && t.requires_grad() ? bit : 0; };
    wants(x, kWantX), wants(residual, kWantResidual), wants(w, kWantWeight), wants(pw, kWantPost), wants(gate, kWantGate);
    if (at::GradMode::is_enabled() && want) return RmsNorm::apply(x, residual_, weight, post, gate_, eps, scale, want);
    Guard guard(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Norms n = norms_forward(x, residual, w, pw, gate, eps, scale, false);
    if (!residual.defined()) return {n.y};
    return {n.y, n.h};
}

// ---------------------------------------------------------------------------------------------- rotary positions
// x [..., heads, dim] as tokens a fixed distance apart
struct Heads {
    Tensor t;
    int64_t tokens = 0, heads = 0, dim = 0, stride = 0, head = 0;
};
Heads heads_of(const Tensor& x) {
    const int64_t n = x.dim();
    Heads r{x, 0, x.size(-2), x.size(-1), 0, 0};
    r.tokens = r.heads && r.dim ? x.numel() / (r.heads * r.dim) : 0;
    bool walks = x.stride(-1) == 1 || r.dim == 1;
    int64_t stride = r.heads * r.dim, size = 1;
    for (int64_t i = n - 3; i >= 0 && walks; --i) {   // dimensions of one element have any stride
        if (x.size(i) == 1) continue;
        if (size == 1) stride = x.stride(i);
        else walks = x.stride(i) == stride * size;
        size *= x.size(i);
    }
    if (!walks) {
        r.t = x.contiguous();
        stride = r.heads * r.dim;
    }
    r.stride = stride;
    r.head = r.heads > 1 ? r.t.stride(-2) : r.dim;
    return r;
}

struct Turn {
    Tensor positions, frequencies;
    bool interleaved;
    double scale;
};
// both outputs, undefined where the input is
std::pair<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Turn& t, bool inverse) {
    std::pair<Tensor, Tensor> out;
    Heads qh, kh;
    ntops_rotary_desc d = {};
    const Tensor& some = q.defined() ? q : k;
    if (q.defined()) {
        out.first = dense_like(q);
        qh = heads_of(q);
        d.q = qh.t.data_ptr(), d.q_out = out.first.data_ptr(), d.q_stride = qh.stride, d.q_head = qh.head, d.heads = (int)qh.heads;
    }
    if (k.defined()) {
        out.second = dense_like(k);
        kh = heads_of(k);
        d.k = kh.t.data_ptr(), d.k_out = out.second.data_ptr(), d.k_stride = kh.stride, d.k_head = kh.head, d.kv_heads = (int)kh.heads;
    }
    d.tokens = q.defined() ? qh.tokens : kh.tokens;
    if (d.tokens == 0) return out;
    d.head_dim = (int)some.size(-1), d.pairs = (int)t.frequencies.numel(), d.dtype = code_of(some, "q");
    d.positions = t.positions.data_ptr(), d.position_count = t.positions.numel(), d.position_bits = t.positions.scalar_type() == at::kLong ? 64 : 32;
    d.frequencies = t.frequencies.const_data_ptr<double>(), d.interleaved = t.interleaved, d.inverse = inverse, d.scale = (float)t.scale;
    call(ntops_rotary(&d, stream_of(some)), "ntops_rotary");
    return out;
}
struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Variable& q, const std::optional<Tensor>& k_, const Tensor& positions, const Tensor& frequencies, bool interleaved, double scale,
                                 bool gq, bool gk) {
        const Tensor k = k_.value_or(Tensor());
        Guard guard(q.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Turn t{positions.contiguous(), frequencies.contiguous(), interleaved, scale};
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({t.positions, t.frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["want"] = (int64_t)(gq | gk << 1);
        ctx->saved_data["type"] = (int64_t)q.scalar_type();
        auto out = rotate(q, k, t, false);
        if (!k.defined()) return {out.first};
        if (!gq) ctx->mark_non_differentiable({out.first});
        if (!gk) ctx->mark_non_differentiable({out.second});
        return {out.first, out.second};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("rotary");
        const variable_list s = ctx->get_saved_variables();
        const int64_t want = ctx->saved_data["want"].toInt();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const auto arrived = [&](size_t i) {
            if (!(want >> i & 1) || i >= grads.size() || !grads[i].defined()) return Tensor();
            return grads[i].scalar_type() == type ? grads[i] : grads[i].to(type);
        };
        const Tensor dq = arrived(0), dk = arrived(1);
        if (!dq.defined() && !dk.defined()) return variable_list(8);
        Guard guard((dq.defined() ? dq : dk).device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Turn t{s[0], s[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble()};
        const auto out = rotate(dq, dk, t, true);
        return {out.first, out.second, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// the rotated q, and k where one is given
std::vector<Tensor> rotary(const Tensor& q, const std::optional<Tensor>& k_, const Tensor& positions, const Tensor& frequencies, bool interleaved, double scale) {
    const Tensor k = k_.value_or(Tensor());
    on_gpu(q, "q");
    code_of(q, "q");
    TORCH_CHECK_VALUE(q.dim() >= 2 && q.size(-1) > 0 && q.size(-2) > 0, "q must have shape [..., heads, head_dim], got ", q.sizes());
    const auto lead = q.sizes().slice(0, q.dim() - 2);
    if (k.defined()) {
        same_device(k, q, "k");
        TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "k must be of the type of q (", q.scalar_type(), "), got ", k.scalar_type());
        TORCH_CHECK_VALUE(k.dim() == q.dim() && k.sizes().slice(0, k.dim() - 2) == lead && k.size(-1) == q.size(-1) && k.size(-2) > 0, "k must have the shape of q but for its heads, ",
                          q.sizes(), ", got ", k.sizes());
    }
    TORCH_CHECK_VALUE(q.size(-1) <= 2048 && q.size(-2) + (k.defined() ? k.size(-2) : 0) <= 16384, "head_dim may be 2048 at most and heads of q and k 16384, got ", q.sizes());
    same_device(positions, q, "positions");
    TORCH_CHECK_TYPE(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "positions must be int64 or int32, got ", positions.scalar_type());
    TORCH_CHECK_VALUE(positions.dim() <= (int64_t)lead.size() && positions.sizes() == lead.slice(lead.size() - positions.dim()),
                      "positions must have the last of the dimensions of q in front of its heads, ", lead, ", got ", positions.sizes());
    same_device(frequencies, q, "frequencies");
    TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kDouble, "frequencies must be float64 (angles of far positions need it), got ", frequencies.scalar_type());
    TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.numel() >= 1 && 2 * frequencies.numel() <= q.size(-1),
                      "frequencies must have shape [pairs], two elements of a head of ", q.size(-1), " each, got ", frequencies.sizes());
    TORCH_CHECK_VALUE(!frequencies.requires_grad(), "frequencies get no gradient: detach them");
    TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
    for (const Tensor* t : {&q, &k}) no_tangent(*t, "rotary");
    const bool gq = q.requires_grad(), gk = k.defined() && k.requires_grad();
    if (at::GradMode::is_enabled() && (gq || gk)) return Rotary::apply(q, k_, positions, frequencies, interleaved, scale, gq, gk);
    Guard guard(q.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const auto out = rotate(q, k, Turn{positions.contiguous(), frequencies.contiguous(), interleaved, scale}, false);
    if (!k.defined()) return {out.first};
    return {out.first, out.second};
}

// ---------------------------------------------------------------------------------------------- attention
// x [rows, heads, dim] or [sequences, rows, heads, dim] as the kernels walk it, copied where they cannot
struct Attended {
    Tensor t;
    int64_t row = 0, head = 0, batch = 0;
};
Attended attended(const Tensor& x) {
    const auto walks = [](const Tensor& t) {
        if (t.numel() == 0) return true;
        const int64_t n = t.dim();
        if (t.stride(n - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
        for (int64_t i = 0; i < n - 1; ++i)
            if (t.size(i) > 1 && (t.stride(i) % 8 != 0 || t.stride(i) < 0 || t.stride(i) > ((int64_t)1 << (i == n - 3 ? 24 : 45)))) return false;
        return true;
    };
    Attended a;
    a.t = walks(x) ? x : x.contiguous();
    if (!walks(a.t)) a.t = a.t.clone(at::MemoryFormat::Contiguous);   // (a dense view that begins off a 16-byte boundary)
    const int64_t n = a.t.dim(), dim = a.t.size(-1);
    // (a dimension of one element, or a tensor of none, may have any distance: nothing walks it)
    const auto stride = [&](int64_t i) { return a.t.size(i) > 1 && a.t.numel() ? a.t.stride(i) : dim; };
    a.head = stride(n - 2), a.row = stride(n - 3), a.batch = n == 4 ? stride(0) : 0;
    return a;
}
struct Sequences {
    Tensor q, k;   // cu_seqlens, or undefined
    double scale;
    bool causal;
};
ntops_attention_desc attention_desc(const Attended& q, const Attended& k, const Attended& v, const Sequences& s) {
    ntops_attention_desc d = {};
    const bool batch = q.t.dim() == 4;
    d.q = q.t.data_ptr(), d.k = k.t.data_ptr(), d.v = v.t.data_ptr();
    d.q_stride = q.row, d.k_stride = k.row, d.v_stride = v.row, d.q_head = q.head, d.k_head = k.head, d.v_head = v.head;
    d.q_batch = q.batch, d.k_batch = k.batch, d.v_batch = v.batch;
    d.heads = (int)q.t.size(-2), d.kv_heads = (int)k.t.size(-2), d.head_dim = (int)q.t.size(-1), d.dtype = code_of(q.t, "q");
    d.sequences = batch ? q.t.size(0) : s.q.defined() ? s.q.numel() - 1 : 1;
    d.q_rows = batch ? q.t.size(0) * q.t.size(1) : q.t.size(0), d.k_rows = batch ? k.t.size(0) * k.t.size(1) : k.t.size(0);
    if (s.q.defined()) d.cu_q = s.q.const_data_ptr<int32_t>(), d.cu_k = s.k.const_data_ptr<int32_t>();
    d.causal = s.causal, d.scale = (float)s.scale;
    return d;
}
Tensor attention_room(ntops_attention_desc& d, bool backward, const Tensor& like) {
    const int64_t bytes = ntops_attention_workspace(&d, backward);
    Tensor ws = at::empty({bytes + 256}, like.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
    d.workspace = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) / 256 * 256);
    return ws;
}
// out, and where a backward pass follows what it needs: lse, the bits that out's rounding left out, and the plan of packed sequences, each on
// a 256-byte boundary
struct AttentionKept {
    int64_t low, plan, bytes;
    explicit AttentionKept(const ntops_attention_desc& d)
        : low((d.heads * d.q_rows * 4 + 255) / 256 * 256), plan(low + (d.heads * d.q_rows * d.head_dim + 255) / 256 * 256), bytes(plan + ntops_attention_plan(&d)) {}
    // (`kept` is 256 bytes longer: a tensor may begin anywhere)
    void into(ntops_attention_desc& d, const Tensor& kept) const {
        char* const at = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(kept.data_ptr()) + 255) / 256 * 256);
        d.lse = reinterpret_cast<float*>(at);
        d.out_low = reinterpret_cast<uint8_t*>(at + low);
        d.plan = d.cu_q ? at + plan : nullptr;
    }
};
std::pair<Tensor, Tensor> attention_forward(const Attended& q, const Attended& k, const Attended& v, const Sequences& s, bool keep) {
    std::pair<Tensor, Tensor> r;
    r.first = dense_like(q.t);
    if (q.t.numel() == 0) return r;
    ntops_attention_desc d = attention_desc(q, k, v, s);
    d.out = r.first.data_ptr();
    if (keep) {
        const AttentionKept room(d);
        r.second = at::empty({room.bytes + 256}, q.t.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
        room.into(d, r.second);
    }
    const Tensor ws = attention_room(d, false, q.t);
    call(ntops_attention_forward(&d, stream_of(q.t)), "ntops_attention_forward");
    return r;
}
struct Attention : torch::autograd::Function<Attention> {
    static Variable forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& v, const std::optional<Tensor>& cu_q, const std::optional<Tensor>& cu_k, bool causal,
                            double scale, bool gq, bool gk, bool gv) {
        Guard guard(q.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Sequences s{contiguous(cu_q.value_or(Tensor())), contiguous(cu_k.value_or(Tensor())), scale, causal};
        const Attended a = attended(q), b = attended(k), c = attended(v);
        const auto r = attention_forward(a, b, c, s, true);
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["want"] = (int64_t)(gq | gk << 1 | gv << 2);
        // (what was copied is kept as the copy)
        ctx->save_for_backward({a.t.is_same(q) ? q : a.t, b.t.is_same(k) ? k : b.t, c.t.is_same(v) ? v : c.t, s.q, s.k, r.first, r.second});
        return r.first;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("attention");
        const variable_list saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return variable_list(10);
        const Variable &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[5];
        Guard guard(q.device());
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t want = ctx->saved_data["want"].toInt();
        Tensor dq, dk, dv;
        if (want & 1) dq = dense_like(q);
        if (want & 2) dk = dense_like(k);
        if (want & 4) dv = dense_like(v);
        const variable_list given = {dq, dk, dv, Variable(), Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
        if (q.numel() == 0 || k.numel() == 0) {   // no pair of a query and a key
            for (Tensor* t : {&dq, &dk, &dv})
                if (t->defined()) t->zero_();
            return given;
        }
        const Sequences s{saved[3], saved[4], ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool()};
        const Attended g = attended(grads[0].scalar_type() == q.scalar_type() ? grads[0] : grads[0].to(q.scalar_type()));
        ntops_attention_desc d = attention_desc(attended(q), attended(k), attended(v), s);
        d.out = out.data_ptr();
        AttentionKept(d).into(d, saved[6]);
        d.dout = g.t.data_ptr(), d.do_stride = g.row, d.do_head = g.head, d.do_batch = g.batch;
        d.dq = at_or_null(dq), d.dk = at_or_null(dk), d.dv = at_or_null(dv);
        const Tensor ws = attention_room(d, true, q);
        call(ntops_attention_backward(&d, stream_of(q)), "ntops_attention_backward");
        return given;
    }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& cu_q, const std::optional<Tensor>& cu_k_, bool causal, const std::optional<double>& scale_) {
    on_gpu(q, "q");
    TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16, got ", q.scalar_type());
    TORCH_CHECK_VALUE(q.dim() == 3 || q.dim() == 4, "q must have shape [tokens, heads, head_dim] or [batch, tokens, heads, head_dim], got ", q.sizes());
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(k, "k"), std::pair<const Tensor&, const char*>(v, "v")}) {
        same_device(t, q, name);
        TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), name, " must be of the type of q (", q.scalar_type(), "), got ", t.scalar_type());
        TORCH_CHECK_VALUE(t.dim() == q.dim() && t.sizes() == k.sizes() && t.size(-1) == q.size(-1) && (q.dim() == 3 || t.size(0) == q.size(0)),
                          "k and v must have one shape, that of q but for tokens and heads: ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
    }
    const int64_t heads = q.size(-2), kv_heads = k.size(-2), dim = q.size(-1);
    TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "the heads of q must be a multiple of those of k, got ", heads, " and ", kv_heads);
    TORCH_CHECK_VALUE(dim > 0 && dim <= 128 && dim % 8 == 0, "head_dim must be a multiple of 8 and 128 at most, got ", dim);
    TORCH_CHECK_VALUE(!cu_k_ || cu_q, "cu_seqlens_k needs cu_seqlens");
    std::optional<Tensor> cu_k = cu_k_;
    if (cu_q) {
        TORCH_CHECK_VALUE(q.dim() == 3, "cu_seqlens goes with packed q of shape [tokens, heads, head_dim], got ", q.sizes());
        if (!cu_k) {
            TORCH_CHECK_VALUE(q.size(0) == k.size(0), "q and k have ", q.size(0), " and ", k.size(0), " tokens: give cu_seqlens_k too");
            cu_k = cu_q;
        }
        for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(*cu_q, "cu_seqlens"), std::pair<const Tensor&, const char*>(*cu_k, "cu_seqlens_k")}) {
            same_device(t, q, name);
            TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
            TORCH_CHECK_VALUE(t.dim() == 1 && t.numel() >= 2 && t.numel() == cu_q->numel(), name, " must have shape [sequences + 1], got ", t.sizes());
        }
    }
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)dim);
    TORCH_CHECK_VALUE(scale >= 1e-30 && scale <= 1e30, "scale must be positive (1e-30 to 1e30), got ", scale);
    for (const Tensor* t : {&q, &k, &v}) no_tangent(*t, "attention");
    const bool gq = q.requires_grad(), gk = k.requires_grad(), gv = v.requires_grad();
    if (at::GradMode::is_enabled() && (gq || gk || gv)) return Attention::apply(q, k, v, cu_q, cu_k, causal, scale, gq, gk, gv);
    Guard guard(q.device());
    at::AutoDispatchBelowADInplaceOrView below;
    return attention_forward(attended(q), attended(k), attended(v), Sequences{contiguous(cu_q.value_or(Tensor())), contiguous(cu_k.value_or(Tensor())), scale, causal}, false).first;
}

// ---------------------------------------------------------------------------------------------- cross entropy
struct Head {
    Tensor loss, losses, dx, dw;
};
// gradients: those asked for, in fp32 where they must still be scaled by something unknown and x is fp16 (its range would not
// hold them), and dw in fp32 where the tokens go in pieces
Head head(const Tensor& x, const Tensor& w, const Tensor& labels, int64_t ignore, bool mean, bool gx, bool gw) {
    const Rows xr = rows_of(x), wr = rows_of(w);
    const Tensor l = labels.contiguous();
    const int xd = code_of(x, "x");
    const auto f32 = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
    ntops_linear_cross_entropy_desc d = {};
    d.tokens = xr.rows, d.hidden = xr.cols, d.vocab = wr.rows, d.x_stride = xr.stride, d.weight_stride = wr.stride;
    d.ignore_index = ignore, d.x_dtype = xd, d.mean = mean;
    d.x = xr.t.data_ptr(), d.weight = wr.t.data_ptr(), d.labels = l.const_data_ptr<int64_t>();
    const bool wide = xd == NTFP8_F16 || (gw && d.tokens > ntops_linear_cross_entropy_piece(d.vocab));
    d.grad_dtype = wide ? NTFP8_F32 : xd;
    Head h;
    const bool gradient = gx || gw;
    if (!gradient) h.losses = at::empty({xr.rows}, f32);
    h.loss = at::empty({}, f32);
    const auto go = wide ? f32 : x.options().memory_format(at::MemoryFormat::Contiguous);
    if (gx) h.dx = at::empty(x.sizes(), go);
    if (gw) h.dw = at::empty(w.sizes(), go);
    d.loss = h.loss.data_ptr<float>(), d.dx = at_or_null(h.dx), d.dweight = at_or_null(h.dw);
    // (with gradients the tokens' losses are nobody's: they lie behind the workspace)
    const int64_t bytes = (ntops_linear_cross_entropy_workspace(&d) + 255) / 256 * 256;
    const Tensor ws = at::empty({256 + bytes + (gradient ? 4 * xr.rows : 0)}, x.options().dtype(at::kByte));
    char* const at = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) / 256 * 256);
    d.workspace = at;
    d.losses = gradient ? reinterpret_cast<float*>(at + bytes) : h.losses.data_ptr<float>();
    call(ntops_linear_cross_entropy(&d, stream_of(x)), "ntops_linear_cross_entropy");
    return h;
}

// The gradients times what arrives from above, of type `to`.  bf16 ones are rounded a second time here unless that is a power of two,
// by 2^-8 of their value at most: held in fp32 until now they would take twice the memory and the way to it.
void scale(Tensor* const (&t)[2], const Tensor& factor, at::ScalarType to) {
    ntops_scale_tensor d[2];
    int n = 0, from = -1;
    for (Tensor* g : t) {
        if (!g->defined()) continue;
        from = code_of(*g, "a gradient");
        const Tensor out = g->scalar_type() == to ? *g : at::empty(g->sizes(), g->options().dtype(to));
        d[n++] = {g->data_ptr(), out.data_ptr(), g->numel()};
        *g = out;
    }
    if (n) call(ntops_scale(d, n, from, factor.const_data_ptr<float>(), to == at::kHalf ? NTFP8_F16 : NTFP8_BF16, stream_of(factor)), "ntops_scale");
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& w, const Variable& labels, int64_t ignore, bool mean, bool gx, bool gw) {
        Guard guard(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        // The gradients are made here, where the softmax is at hand, and scaled by what arrives in backward, so that nothing of
        // the logits' size outlives this call
        Head h = head(x, w, labels, ignore, mean, gx, gw);
        ctx->saved_data["dx"] = h.dx;
        ctx->saved_data["dw"] = h.dw;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        return h.loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("linear_cross_entropy");
        TORCH_CHECK(ctx->saved_data.count("type"),
                    "linear_cross_entropy: its gradients are handed over once and not kept; compute the loss again for another backward pass");
        Tensor dx, dw;
        if (ctx->saved_data["dx"].isTensor()) dx = ctx->saved_data["dx"].toTensor();
        if (ctx->saved_data["dw"].isTensor()) dw = ctx->saved_data["dw"].toTensor();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        ctx->saved_data.clear();
        if (!grads[0].defined()) return variable_list(7);
        Guard guard(grads[0].device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = grads[0].to(at::kFloat);
        const Tensor held_dx = dx, held_dw = dw;   // (until the launch that reads them is queued)
        scale({&dx, &dw}, g, type);
        return {dx, dw, Variable(), Variable(), Variable(), Variable(), Variable()};
    }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& w, const Tensor& labels, int64_t ignore, const std::string& reduction) {
    on_gpu(x, "x");
    same_device(w, x, "weight");
    same_device(labels, x, "labels");
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type(), "weight must be of the type of x (", x.scalar_type(), "), got ", w.scalar_type());
    TORCH_CHECK_TYPE(labels.scalar_type() == at::kLong, "labels must be int64, got ", labels.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && w.size(0) > 0 && w.size(1) > 0 && x.size(-1) == w.size(1), "x [..., hidden] and weight [vocab, hidden] do not fit: ", x.sizes(),
                      " and ", w.sizes());
    TORCH_CHECK_VALUE(labels.sizes() == x.sizes().slice(0, x.dim() - 1), "labels must have the shape of x without its last dimension, got ", labels.sizes(), " for x ", x.sizes());
    const bool mean = reduction == "mean", none = reduction == "none";
    TORCH_CHECK_VALUE(mean || none || reduction == "sum", "reduction must be 'mean', 'sum' or 'none', got '", reduction, "'");
    const bool gx = x.requires_grad(), gw = w.requires_grad(), wants = at::GradMode::is_enabled() && (gx || gw);
    TORCH_CHECK_VALUE(!(none && wants), "reduction='none' gives the losses of single tokens without gradients: call it under torch.no_grad()");
    for (const Tensor* t : {&x, &w}) no_tangent(*t, "linear_cross_entropy");
    if (x.numel() == 0) {   // no tokens: a loss of 0 without gradient
        const auto f32 = x.options().dtype(at::kFloat);
        return none ? at::zeros(labels.sizes(), f32) : (x.sum() + w.narrow(0, 0, 0).sum()).to(at::kFloat);
    }
    if (wants) return LinearCrossEntropy::apply(x, w, labels, ignore, mean, gx, gw);
    Guard guard(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Head h = head(x, w, labels, ignore, mean, false, false);
    return none ? h.losses.view(labels.sizes()) : h.loss;
}

// ---------------------------------------------------------------------------------------------- AdamW
// A list or tuple of tensors as the objects that it holds: hundreds of them come in every step, and as a vector of tensors each
// would cost a reference more
struct List {
    py::object own;
    PyObject** items = nullptr;
    size_t n = 0;
    explicit List(const py::object& o, const char* name) {
        if (o.is_none()) return;
        own = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "a list of tensors is expected"));
        if (!own) throw py::error_already_set();
        items = PySequence_Fast_ITEMS(own.ptr());
        n = (size_t)PySequence_Fast_GET_SIZE(own.ptr());
        for (size_t i = 0; i < n; ++i) TORCH_CHECK_TYPE(items[i] == Py_None || THPVariable_Check(items[i]), name, " must be a list of tensors");
    }
    bool given() const { return items != nullptr || own; }
    bool none(size_t i) const { return items[i] == Py_None; }
    const Tensor& operator[](size_t i) const {
        TORCH_CHECK_TYPE(items[i] != Py_None, "a tensor is expected, got None");
        return THPVariable_Unpack(items[i]);
    }
};

void adamw(const py::object& params_, const py::object& grads_, const py::object& m_, const py::object& v_, const py::object& ms_, const py::object& vs_,
           const py::object& copies_, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step, int64_t seed, const std::optional<Tensor>& grad_scale) {
    const List params(params_, "params"), grads(grads_, "grads"), m(m_, "first moments"), v(v_, "second moments"), ms(ms_, "scales"), vs(vs_, "scales"), copies(copies_, "copies");
    const size_t n = params.n;
    const bool small = ms.given();
    TORCH_CHECK_VALUE(grads.n == n && m.n == n && v.n == n && (!small || (ms.n == n && vs.n == n)) && (!copies.given() || copies.n == n),
                      "the lists of an AdamW step must have one length (", n, " parameters)");
    TORCH_CHECK_VALUE(step >= 1, "step counts from 1, got ", step);
    TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must lie in [0, 1), got ", beta1, " and ", beta2);
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
    if (n == 0) return;
    const Tensor& p0 = params[0];
    on_gpu(p0, "a parameter");
    const c10::Device device = p0.device();
    Guard guard(device);
    ntops_adamw_options o = {};
    o.lr = lr, o.beta1 = beta1, o.beta2 = beta2, o.eps = eps, o.weight_decay = weight_decay, o.step = step, o.seed = (uint32_t)seed, o.bits = small ? 8 : 32;
    if (grad_scale) {
        same_device(*grad_scale, p0, "grad_scale");
        TORCH_CHECK_TYPE(grad_scale->scalar_type() == at::kFloat && grad_scale->numel() == 1, "grad_scale must be one float32 value");
        o.grad_scale = grad_scale->const_data_ptr<float>();
    }
    // one call for each set of types, in the order in which they first come
    struct Kind {
        int p, g, c;
        std::vector<ntops_adamw_tensor> t;
    };
    std::vector<Kind> kinds;
    const auto state = small ? at::kByte : at::kFloat;
    for (size_t i = 0; i < n; ++i) {
        const Tensor& p = params[i];
        const int64_t count = p.numel();
        auto fits = [&](const Tensor& t, const char* name, int64_t want) -> void* {
            if (C10_UNLIKELY(t.device() != device || t.numel() != want || !t.is_contiguous())) {
                same_device(t, p0, name);
                TORCH_CHECK_VALUE(false, name, " ", i, " must be contiguous with ", want, " elements, got shape ", t.sizes(), " and strides ", t.strides());
            }
            return t.data_ptr();
        };
        ntops_adamw_tensor t = {};
        t.param = fits(p, "parameter", count), t.grad = fits(grads[i], "gradient", count), t.exp_avg = fits(m[i], "first moment", count);
        t.exp_avg_sq = fits(v[i], "second moment", count), t.n = count;
        TORCH_CHECK_TYPE(m[i].scalar_type() == state && v[i].scalar_type() == state, "moments must be ", state, ", got ", m[i].scalar_type(), " and ", v[i].scalar_type());
        if (small) {
            const int64_t blocks = (count + NTOPS_ADAMW_BLOCK - 1) / NTOPS_ADAMW_BLOCK;
            TORCH_CHECK_TYPE(ms[i].scalar_type() == at::kFloat && vs[i].scalar_type() == at::kFloat, "scales of moments must be float32");
            t.exp_avg_scale = static_cast<float*>(fits(ms[i], "scales of the first moment", blocks));
            t.exp_avg_sq_scale = static_cast<float*>(fits(vs[i], "scales of the second moment", blocks));
        }
        const int pc = code_of(p, "a parameter"), gc = code_of(grads[i], "a gradient");
        int cc = -1;
        if (copies.given() && !copies.none(i)) {
            t.copy = fits(copies[i], "copy", count);
            cc = code_of(copies[i], "a copy");
        }
        auto at = std::find_if(kinds.begin(), kinds.end(), [&](const Kind& q) { return q.p == pc && q.g == gc && q.c == cc; });
        if (at == kinds.end()) {
            at = kinds.insert(kinds.end(), Kind{pc, gc, cc, {}});
            at->t.reserve(n - i);
        }
        at->t.push_back(t);
    }
    // all sets are looked over before the first is launched: a step that is refused has changed nothing
    const auto each = [&](auto&& f) {
        for (const Kind& k : kinds) {
            o.param_dtype = k.p, o.grad_dtype = k.g, o.copy_dtype = k.c;
            call(f(k.t.data(), (int)k.t.size()), "ntops_adamw");
        }
    };
    if (kinds.size() > 1) each([&](const ntops_adamw_tensor* t, int count) { return ntops_adamw_check(t, count, &o); });
    each([&](const ntops_adamw_tensor* t, int count) { return ntops_adamw(t, count, &o, stream_of(p0)); });
    // (autograd's record of in-place changes: a graph that saved a parameter or its copy finds out)
    const auto changed = [](const Tensor& t) {
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    for (size_t i = 0; i < n; ++i) {
        changed(params[i]);
        if (copies.given() && !copies.none(i)) changed(copies[i]);
    }
}

Tensor adamw_unpack(const Tensor& codes, const Tensor& scale) {
    on_gpu(codes, "codes");
    same_device(scale, codes, "scale");
    TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scale.scalar_type() == at::kFloat, "codes must be uint8 and scale float32");
    TORCH_CHECK_VALUE(codes.is_contiguous() && scale.is_contiguous() && scale.numel() == (codes.numel() + NTOPS_ADAMW_BLOCK - 1) / NTOPS_ADAMW_BLOCK,
                      "scale must hold one value for every ", NTOPS_ADAMW_BLOCK, " codes");
    Guard guard(codes.device());
    Tensor out = at::empty(codes.sizes(), codes.options().dtype(at::kFloat));
    if (codes.numel()) call(ntops_adamw_unpack(codes.data_ptr(), scale.const_data_ptr<float>(), codes.numel(), out.data_ptr<float>(), stream_of(codes)), "ntops_adamw_unpack");
    return out;
}

}  // namespace

PYBIND11_MODULE(_opscall, m) {
    m.def("layer_norm", &layer_norm);
    m.def("rms_norm", &rms_norm);
    m.def("rotary", &rotary);
    m.def("attention", &attention);
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("adamw", &adamw);
    m.def("adamw_unpack", &adamw_unpack);
}
