// The host side of the operators of a transformer block around its attention (include/bptblock.h), part of bptop.so: checks,
// allocation, launches and autograd without the interpreter.  They have no plans: a call is checked and launched, nothing is kept.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <tuple>

#include "../../include/bptattn.h"
#include "../../include/bptblock.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

using Optional = std::optional<Tensor>;

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_status(int st, const char *what) { TORCH_CHECK(st == BPT_OK, what, ": ", bpt_strerror(st), " (status ", st, ")"); }

void check_input(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided && t.is_contiguous(), name, " must be contiguous");
}
void check_like(const Tensor &t, const Tensor &x, const char *name) {
    check_input(t, name);
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), "all floating point arguments must share one dtype");
    TORCH_CHECK_VALUE(t.device() == x.device(), "all tensors of a call must be on one device");
}
void check_shape(const Tensor &t, at::IntArrayRef shape, const char *name) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}

int dtype_code(const Tensor &t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? BPT_F32 : s == at::kBFloat16 ? BPT_BF16 : s == at::kDouble ? BPT_F64 : -1;
}

bool differentiated(std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
        if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
    return false;
}

void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// ---- layer norm of a sum ------------------------------------------------------------------------------------------------------
void check_norm(const Tensor &x, const Tensor &r, const Tensor &w, const Tensor &b, double eps) {
    check_input(x, "x");
    TORCH_CHECK(dtype_code(x) >= 0, "unsupported dtype ", x.scalar_type(), ": float32, float64 and bfloat16 are implemented");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last axis of one element at least");
    TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative");
    if (r.defined()) {
        check_like(r, x, "residual");
        check_shape(r, x.sizes(), "residual");
    }
    for (const auto &[t, name] : {std::pair<const Tensor &, const char *>{w, "weight"}, {b, "bias"}})
        if (t.defined()) {
            check_like(t, x, name);
            check_shape(t, {x.size(-1)}, name);
        }
}

int64_t rows_of(const Tensor &x) { return x.numel() / x.size(-1); }

std::tuple<Tensor, Tensor> norm_forward(const Tensor &x, const Tensor &r, const Tensor &w, const Tensor &b, double eps, bool keep) {
    c10::DeviceGuard guard(x.device());
    const int64_t rows = rows_of(x);
    Tensor y = at::empty_like(x), stats;
    if (keep) stats = at::empty({rows, 2}, x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat));
    check_status(bpt_add_norm_forward(ptr(x), ptr(r), ptr(w), ptr(b), ptr(y), ptr(stats), rows, x.size(-1), eps, dtype_code(x), stream_of(x)), "add_layer_norm");
    return {y, stats};
}

struct AddLayerNorm : torch::autograd::Function<AddLayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Optional &residual, const Optional &weight, const Optional &bias, double eps) {
        const Tensor r = residual.value_or(Tensor()), w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        const auto [y, stats] = norm_forward(x, r, w, b, eps, true);
        ctx->save_for_backward({x, r, w, b, stats});
        ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto t = ctx->get_saved_variables();
        const Tensor &x = t[0], &r = t[1], &w = t[2], &b = t[3], &stats = t[4];
        size_t edge = 0;                                          // (counted over the arguments that are tensors)
        auto needed = [&](const Tensor &arg) { return arg.defined() && ctx->needs_input_grad(edge++); };
        const bool need_x = needed(x), need_r = needed(r), need_w = needed(w), need_b = needed(b), need_z = need_x || need_r;
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        if (at::GradMode::is_enabled()) {
            // a gradient that is to be differentiated again: in operations that can be
            const Tensor z = r.defined() ? x + r : x;
            const auto [y, mean, rstd] = at::native_layer_norm(z, {x.size(-1)}, w, b, ctx->saved_data["eps"].toDouble());
            const auto [dz, dw, db] = at::native_layer_norm_backward(grads[0], z, {x.size(-1)}, mean, rstd, w, b, {need_z, need_w, need_b});
            return {need_x ? dz : Tensor(), need_r ? dz : Tensor(), dw, db, Tensor()};
        }
        // (the saved tensors may be others than the forward's: a hook on them can give back anything)
        check_norm(x, r, w, b, 0.0);
        const int64_t rows = rows_of(x), cols = x.size(-1);
        TORCH_CHECK(stats.is_cuda() && stats.is_contiguous() && stats.dim() == 2 && stats.size(0) == rows && stats.size(1) == 2 && stats.device() == x.device() &&
                        stats.scalar_type() == (x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat),
                    "stats must be the tensor that the forward saved");
        const Tensor dy = grads[0].contiguous();
        check_like(dy, x, "dy");
        check_shape(dy, x.sizes(), "dy");
        c10::DeviceGuard guard(x.device());
        Tensor dz, dw, db, ws;
        if (need_z) dz = at::empty_like(x);
        if (need_w) dw = at::empty_like(w);
        if (need_b) db = at::empty_like(b);
        const int64_t bytes = need_w || need_b ? bpt_add_norm_workspace_bytes(rows, cols, dtype_code(x)) : 0;
        if (bytes > 0) ws = at::empty({bytes}, x.options().dtype(at::kByte));
        check_status(bpt_add_norm_backward(ptr(x), ptr(r), ptr(w), ptr(stats), ptr(dy), ptr(dz), ptr(dw), ptr(db), ptr(ws), bytes, rows, cols, dtype_code(x),
                                           stream_of(x)),
                     "add_layer_norm's backward");
        return {need_x ? dz : Tensor(), need_r ? dz : Tensor(), dw, db, Tensor()};
    }
};

Tensor add_layer_norm(const Tensor &x, const Optional &residual, const Optional &weight, const Optional &bias, double eps) {
    const Tensor r = residual.value_or(Tensor()), w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    check_norm(x, r, w, b, eps);
    if (differentiated({&x, &r, &w, &b})) return AddLayerNorm::apply(x, residual, weight, bias, eps);
    return std::get<0>(norm_forward(x, r, w, b, eps, false));
}

// ---- relu kept in 8 bits -----------------------------------------------------------------------------------------------------
void check_relu8(const Tensor &a, double p, const char *name) {
    check_input(a, name);
    const int dt = dtype_code(a);
    TORCH_CHECK(dt == BPT_F32 || dt == BPT_BF16, "unsupported dtype ", a.scalar_type(), ": float32 and bfloat16 are implemented");
    TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "dropout_p must be in [0, 1)");
}

using Three = std::tuple<Tensor, Tensor, Tensor>;

Three relu8_forward(const Tensor &a, double p, uint64_t seed) {
    check_relu8(a, p, "a");
    c10::DeviceGuard guard(a.device());
    Tensor y = at::empty_like(a), codes = at::empty_like(a, a.options().dtype(at::kByte));
    Tensor exps = at::empty({(a.numel() + BPT_RELU8_BLOCK - 1) / BPT_RELU8_BLOCK}, a.options().dtype(at::kChar));
    check_status(bpt_relu8_forward(ptr(a), ptr(y), (uint8_t *)ptr(codes), (int8_t *)ptr(exps), a.numel(), (float)p, seed, dtype_code(a), stream_of(a)),
                 "relu8_forward");
    return {y, codes, exps};
}

// the codes and exponents of a gradient like dy
void check_codes(const Tensor &codes, const Tensor &exps, const Tensor &dy) {
    check_input(codes, "codes");
    check_input(exps, "exps");
    TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && exps.scalar_type() == at::kChar, "codes must be uint8 and exps int8, as relu8_forward returns them");
    TORCH_CHECK_VALUE(codes.device() == dy.device() && exps.device() == dy.device(), "all tensors of a call must be on one device");
    check_shape(codes, dy.sizes(), "codes");
    check_shape(exps, {(dy.numel() + BPT_RELU8_BLOCK - 1) / BPT_RELU8_BLOCK}, "exps");
}

// into: null, or the tensor that receives da (dy itself, where nobody else has it)
std::tuple<Tensor, Tensor> relu8_backward_into(const Tensor &dy, const Tensor &codes, const Tensor &exps, double p, const Tensor &into) {
    check_relu8(dy, p, "dy");
    check_codes(codes, exps, dy);
    c10::DeviceGuard guard(dy.device());
    Tensor da = into.defined() ? into : at::empty_like(dy), y8 = at::empty_like(dy);
    check_status(bpt_relu8_backward(ptr(dy), (const uint8_t *)ptr(codes), (const int8_t *)ptr(exps), ptr(da), ptr(y8), dy.numel(), (float)p, dtype_code(dy),
                                    stream_of(dy)),
                 "relu8_backward");
    return {da, y8};
}
// what the codes stand for, in y8
void relu8_values(const Tensor &codes, const Tensor &exps, Tensor &y8) {
    check_codes(codes, exps, y8);
    c10::DeviceGuard guard(y8.device());
    check_status(bpt_relu8_backward(nullptr, (const uint8_t *)ptr(codes), (const int8_t *)ptr(exps), nullptr, ptr(y8), y8.numel(), 0.f, dtype_code(y8), stream_of(y8)),
                 "relu8_backward");
}
std::tuple<Tensor, Tensor> relu8_backward(const Tensor &dy, const Tensor &codes, const Tensor &exps, double p) {
    return relu8_backward_into(dy, codes, exps, p, Tensor());
}

void check_relu_linear(const Tensor &a, const Tensor &w, const Tensor &b, double p) {
    check_relu8(a, p, "a");
    TORCH_CHECK_VALUE(a.dim() >= 1 && a.size(-1) >= 1, "a must have a last axis of one element at least");
    check_like(w, a, "weight");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == a.size(-1), "weight must be (outputs, ", a.size(-1), "), got ", w.sizes());
    if (b.defined()) {
        check_like(b, a, "bias");
        check_shape(b, {w.size(0)}, "bias");
    }
}

// the products are of the tensors as they are, also inside autocast (whose results the backward would meet in another type)
using NoAutocast = c10::impl::ExcludeDispatchKeyGuard;

struct ReluLinear8 : torch::autograd::Function<ReluLinear8> {
    static Tensor forward(AutogradContext *ctx, const Tensor &a, const Tensor &w, const Optional &b, double p, int64_t seed) {
        const NoAutocast as_it_is(c10::DispatchKey::AutocastCUDA);
        const auto [y, codes, exps] = relu8_forward(a, p, (uint64_t)seed);
        ctx->save_for_backward({codes, exps, w});
        ctx->saved_data["p"] = p;
        ctx->saved_data["bias"] = b.has_value();
        return at::linear(y, w, b);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "relu_linear8 is not differentiable twice");
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        const NoAutocast as_it_is(c10::DispatchKey::AutocastCUDA);
        const auto t = ctx->get_saved_variables();
        const Tensor &codes = t[0], &exps = t[1], &w = t[2];
        const double p = ctx->saved_data["p"].toDouble();
        const bool need_a = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
        const int64_t inner = w.size(1), outer = w.size(0), rows = inner ? codes.numel() / inner : 0;
        const Tensor d_o = grads[0].contiguous().view({rows, outer});
        Tensor da, dw, db;
        if (need_a) {
            const Tensor dy = at::mm(d_o, w);
            const auto [d, y8] = relu8_backward_into(dy, codes.view({rows, inner}), exps, p, dy);
            da = d.view(codes.sizes());
            if (need_w) dw = at::mm(d_o.t(), y8);
        } else if (need_w) {                                      // (nobody reads dy, so nobody forms it)
            Tensor y8 = at::empty({rows, inner}, d_o.options());
            relu8_values(codes.view({rows, inner}), exps, y8);
            dw = at::mm(d_o.t(), y8);
        }
        if (need_b) {                                             // (the column sums of the layer norm's backward)
            c10::DeviceGuard guard(d_o.device());
            db = at::empty({outer}, d_o.options());
            if (outer == 0) return {da, dw, db, Tensor(), Tensor()};
            const int64_t bytes = bpt_add_norm_workspace_bytes(rows, outer, dtype_code(d_o));
            const Tensor ws = at::empty({bytes}, d_o.options().dtype(at::kByte));
            check_status(bpt_add_norm_backward(ptr(d_o), nullptr, nullptr, nullptr, ptr(d_o), nullptr, nullptr, ptr(db), ptr(ws), bytes, rows, outer,
                                               dtype_code(d_o), stream_of(d_o)),
                         "relu_linear8's backward");
        }
        return {da, dw, db, Tensor(), Tensor()};
    }
};

Tensor relu_linear8(const Tensor &a, const Tensor &weight, const Optional &bias, double p, uint64_t seed) {
    const Tensor b = bias.value_or(Tensor());
    check_relu_linear(a, weight, b, p);
    if (differentiated({&a, &weight, &b})) return ReluLinear8::apply(a, weight, bias, p, (int64_t)seed);
    const NoAutocast as_it_is(c10::DispatchKey::AutocastCUDA);
    if (p == 0.0) return at::linear(at::relu(a), weight, bias);     // (nothing to keep)
    return at::linear(std::get<0>(relu8_forward(a, p, seed)), weight, bias);
}

}  // namespace

void bind_block(py::module_ &m) {
    m.def("add_layer_norm", &add_layer_norm);
    m.def("relu8_forward", &relu8_forward);
    m.def("relu8_backward", &relu8_backward);
    m.def("relu_linear8", &relu_linear8);
}
