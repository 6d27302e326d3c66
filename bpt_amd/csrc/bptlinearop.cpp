// The host side of matrix products with an epilogue and of dropout (include/bptlinear.h), part of bptop.so: checks, allocation, launches and
// autograd without the interpreter.  Nothing is kept from call to call.
#include "bpthost.h"

#include "../../include/bptlinear.h"

namespace {

Tensor workspace(int64_t bytes, const Tensor &like) { return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }

void check_type(const Tensor &x, const char *name) {
    check_input(x, name);
    const int dt = dtype_code(x);
    TORCH_CHECK(dt == BPT_F32 || dt == BPT_BF16, "unsupported dtype ", x.scalar_type(), ": float32 and bfloat16 are implemented");
}
void check_share(double p) { TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "dropout_p must be in [0, 1)"); }

// ---- matrix products with an epilogue ------------------------------------------------------------------------------------------
struct Sizes {
    int64_t rows, inner, outer;
    std::vector<int64_t> shape;                  // of the result
};
Sizes check_linear(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, int64_t act, double p) {
    check_type(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last axis of one element at least");
    check_like(w, x, "weight");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1), "weight must be (outputs, ", x.size(-1), "), got ", w.sizes());
    Sizes n{x.numel() / x.size(-1), x.size(-1), w.size(0), x.sizes().vec()};
    n.shape.back() = n.outer;
    if (b.defined()) {
        check_like(b, x, "bias");
        check_shape(b, {n.outer}, "bias");
    }
    if (r.defined()) {
        check_like(r, x, "residual");
        check_shape(r, n.shape, "residual");
    }
    TORCH_CHECK_VALUE(act >= BPT_ACT_NONE && act <= BPT_ACT_GELU, "unknown activation");
    check_share(p);
    return n;
}

// (y, a where it is to be kept)
std::tuple<Tensor, Tensor> linear_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, int64_t act, double p, uint64_t seed, bool keep) {
    const Sizes n = check_linear(x, w, b, r, act, p);
    c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(n.shape, x.options()), kept;
    if (keep) kept = at::empty_like(y);
    const int dt = dtype_code(x);
    const int64_t bytes = bpt_linear_forward_workspace_bytes(n.rows, n.inner, n.outer, dt);
    const Tensor ws = workspace(bytes, x);
    check_status(bpt_linear_forward(ptr(x), ptr(w), ptr(b), ptr(r), ptr(y), ptr(kept), ptr(ws), bytes, n.rows, n.inner, n.outer, (int)act, p, seed, dt, stream_of(x)),
                 "linear_act");
    return {y, kept};
}

struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Optional &bias, const Optional &residual, int64_t act, double p, int64_t seed) {
        const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
        // relu's result tells where it let through what dropout kept, unless a residual was added to it; otherwise a is kept
        const bool products = x.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad());
        const bool result = products && act == BPT_ACT_RELU && !r.defined(), keep = products && act != BPT_ACT_NONE && !result;
        const auto [y, kept] = linear_forward(x, w, b, r, act, p, (uint64_t)seed, keep);
        ctx->save_for_backward({x, w, result ? y : kept});
        ctx->saved_data["act"] = act;
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["result"] = result;
        ctx->saved_data["bias"] = b.defined();
        ctx->saved_data["residual"] = r.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_act is not differentiable twice");
        if (!grads[0].defined()) return variable_list(7);
        const auto t = ctx->get_saved_variables();
        const Tensor &x = t[0], &w = t[1], &kept = t[2];
        const int64_t act = ctx->saved_data["act"].toInt();
        const double p = ctx->saved_data["p"].toDouble();
        const uint64_t seed = (uint64_t)ctx->saved_data["seed"].toInt();
        const bool result = ctx->saved_data["result"].toBool(), has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
        size_t edge = 0;                                          // (counted over the arguments that are tensors)
        auto needed = [&](bool given) { return given && ctx->needs_input_grad(edge++); };
        const bool need_x = needed(true), need_w = needed(true), need_b = needed(has_b), need_r = needed(has_r);
        variable_list out(7);
        if (need_r) out[3] = grads[0];
        if (!need_x && !need_w && !need_b) return out;
        // (the saved tensors may be others than the forward's: a hook on them can give back anything)
        const Sizes n = check_linear(x, w, Tensor(), Tensor(), act, p);
        const Tensor dy = grads[0].contiguous();
        check_like(dy, x, "dy");
        check_shape(dy, n.shape, "dy");
        if (act != BPT_ACT_NONE) {
            TORCH_CHECK(kept.defined(), "what the forward kept is missing");
            check_like(kept, x, "kept");
            check_shape(kept, n.shape, "kept");
        }
        c10::DeviceGuard guard(x.device());
        const int dt = dtype_code(x);
        void *const stream = stream_of(x);
        const double scale = 1.0 / (1.0 - p);
        Tensor g = dy;
        const bool changes = act != BPT_ACT_NONE || p > 0.0;
        if (changes && (need_x || need_w)) g = at::empty_like(dy);
        if (need_b) out[2] = at::empty({n.outer}, x.options());
        if (changes || need_b) {
            const int64_t bytes = need_b ? bpt_linear_grad_workspace_bytes(n.rows, n.outer, dt) : 0;
            const Tensor ws = workspace(bytes, x);
            check_status(bpt_linear_grad(ptr(dy), ptr(kept), result, changes && (need_x || need_w) ? ptr(g) : nullptr, ptr(out[2]), ptr(ws), bytes, n.rows, n.outer,
                                         (int)act, p, seed, dt, stream),
                         "linear_act's backward");
        }
        if (need_x) {
            out[0] = n.outer == 0 ? at::zeros_like(x) : at::empty_like(x);
            if (n.outer > 0) {
                const int64_t bytes = bpt_linear_input_grad_workspace_bytes(n.rows, n.inner, n.outer, dt);
                const Tensor ws = workspace(bytes, x);
                check_status(bpt_linear_input_grad(ptr(g), ptr(w), ptr(out[0]), ptr(ws), bytes, n.rows, n.inner, n.outer, scale, dt, stream), "linear_act's backward");
            }
        }
        if (need_w) {
            out[1] = n.rows == 0 ? at::zeros_like(w) : at::empty_like(w);
            if (n.rows > 0) {
                const int64_t bytes = bpt_linear_weight_grad_workspace_bytes(n.rows, n.inner, n.outer, dt);
                const Tensor ws = workspace(bytes, x);
                check_status(bpt_linear_weight_grad(ptr(g), ptr(x), ptr(out[1]), ptr(ws), bytes, n.rows, n.inner, n.outer, scale, dt, stream), "linear_act's backward");
            }
        }
        return out;
    }
};

Tensor linear_act(const Tensor &x, const Tensor &weight, const Optional &bias, const Optional &residual, int64_t act, double p, uint64_t seed) {
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    if (differentiated({&x, &weight, &b, &r})) {
        check_linear(x, weight, b, r, act, p);
        return LinearAct::apply(x, weight, bias, residual, act, p, (int64_t)seed);
    }
    return std::get<0>(linear_forward(x, weight, b, r, act, p, seed, false));
}

// ---- dropout -----------------------------------------------------------------------------------------------------------------------
Tensor dropout_call(const Tensor &x, const Tensor &r, double p, uint64_t seed) {
    check_type(x, "x");
    check_share(p);
    if (r.defined()) {
        check_like(r, x, "residual");
        check_shape(r, x.sizes(), "residual");
    }
    c10::DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x);
    check_status(bpt_dropout(ptr(x), ptr(r), ptr(y), x.numel(), p, seed, dtype_code(x), stream_of(x)), "dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Optional &residual, double p, int64_t seed) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["residual"] = residual.has_value();
        return dropout_call(x, residual.value_or(Tensor()), p, (uint64_t)seed);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const double p = ctx->saved_data["p"].toDouble();
        const int64_t seed = ctx->saved_data["seed"].toInt();
        if (ctx->needs_input_grad(0)) {
            const Tensor dy = grads[0].contiguous();
            // (a gradient that is to be differentiated again is a dropout of its own)
            out[0] = at::GradMode::is_enabled() && dy.requires_grad() ? Dropout::apply(dy, std::nullopt, p, seed) : dropout_call(dy, Tensor(), p, (uint64_t)seed);
        }
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
        return out;
    }
};

Tensor dropout(const Tensor &x, const Optional &residual, double p, uint64_t seed) {
    const Tensor r = residual.value_or(Tensor());
    if (differentiated({&x, &r})) return Dropout::apply(x, residual, p, (int64_t)seed);
    return dropout_call(x, r, p, seed);
}

}  // namespace

void bind_linear(py::module_ &m) {
    m.def("linear_act", &linear_act);
    m.def("dropout", &dropout);
}
