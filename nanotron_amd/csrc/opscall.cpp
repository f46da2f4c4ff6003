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
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("adamw", &adamw);
    m.def("adamw_unpack", &adamw_unpack);
}
