// gated_scan and linear8 as autograd functions. On the host side a small call is
// all overhead: a Python autograd function costs some 60 us for forward and
// backward, this one under a third of it.
#include <torch/extension.h>

#include <c10/core/impl/LocalDispatchKeySet.h>

#include "launchers.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kEvery = 16;  // tokens between two kept states
constexpr int64_t kGroup = 32;  // values that share a scale

c10::optional<Tensor> some(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }

void first_order(const char* what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient has no gradient of its own (create_graph)");
}

bool dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

struct Scan {
    Tensor y, last, states, codes, scales;
};

Scan scan(const Tensor& p, int64_t dim, const c10::optional<Tensor>& h0, const c10::optional<Tensor>& lengths,
          bool train, bool keep8) {
    const int64_t B = p.size(0), T = p.size(1);
    const auto f32 = p.options().dtype(at::kFloat);
    Scan s;
    s.y = at::empty({B, T, dim}, p.options());
    s.last = at::empty({B, dim}, f32);
    if (train) s.states = at::empty({B, (T + kEvery - 1) / kEvery, dim}, f32);
    if (keep8) {
        const int64_t rows = B * T * (p.size(2) / dim), groups = (dim + kGroup - 1) / kGroup;
        s.codes = at::empty({rows, groups * kGroup}, p.options().dtype(at::kChar));
        s.scales = at::empty({B, (T + kEvery - 1) / kEvery, p.size(2) / dim, groups, kEvery}, p.options().dtype(at::kByte));
    }
    gated_scan_fwd_launch(p, dim, h0, lengths, s.y, s.last, some(s.states), some(s.codes), some(s.scales));
    return s;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& p, const c10::optional<Tensor>& h0,
                                 const c10::optional<Tensor>& lengths, int64_t dim, bool keep8) {
        Scan s = scan(p, dim, h0, lengths, true, keep8);
        ctx->saved_data["dim"] = dim;
        ctx->saved_data["h0"] = h0.has_value() && h0->requires_grad();
        ctx->saved_data["width"] = p.size(2);
        ctx->save_for_backward({keep8 ? Tensor() : p, lengths.value_or(Tensor()), s.states, s.codes, s.scales});
        return {s.y, s.last};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_order("gated_scan");
        const auto saved = ctx->get_saved_variables();
        const Tensor &p = saved[0], &states = saved[2], &codes = saved[3];
        const int64_t dim = ctx->saved_data["dim"].toInt(), width = ctx->saved_data["width"].toInt();
        Tensor dy = grads[0], dh = grads[1].contiguous();
        if (dim > 1 && dy.stride(2) != 1) dy = dy.contiguous();
        Tensor dp = at::empty({dy.size(0), dy.size(1), width}, dy.options());
        Tensor dh0 = ctx->saved_data["h0"].toBool() ? at::empty_like(dh) : Tensor();
        // with codes the projection itself is gone; dp stands in for its shape
        gated_scan_bwd_launch(codes.defined() ? dp : p, dim, some(saved[1]), states, some(codes), some(saved[4]), dy, dh, dp, some(dh0));
        return {dp, dh0, Tensor(), Tensor(), Tensor()};
    }
};

Tensor project(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias) {
    const auto type = x.scalar_type();
    return at::linear(x, weight.to(type), bias.has_value() ? c10::optional<Tensor>(bias->to(type)) : c10::nullopt);
}

struct Linear8 : torch::autograd::Function<Linear8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias) {
        const Tensor y = project(x, weight, bias);
        Tensor codes, scales;
        if (weight.requires_grad()) {
            const int64_t F = x.size(-1);
            Tensor rows = x.reshape({x.numel() / F, F});
            if (F > 1 && rows.stride(1) != 1) rows = rows.contiguous();
            std::tie(codes, scales) = save8_launch(rows);
        }
        ctx->saved_data["x"] = x.requires_grad();
        ctx->saved_data["bias"] = bias.has_value() && bias->requires_grad();
        ctx->saved_data["bias_type"] = (int64_t)(bias.has_value() ? bias->scalar_type() : weight.scalar_type());
        ctx->save_for_backward({weight, codes, scales});
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_order("linear8");
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        const auto saved = ctx->get_saved_variables();
        const Tensor &weight = saved[0], &codes = saved[1], &dy = grads[0];
        const bool bias = ctx->saved_data["bias"].toBool();
        const auto bias_type = (at::ScalarType)ctx->saved_data["bias_type"].toInt();
        Tensor dx, dw, db;
        if (ctx->saved_data["x"].toBool()) dx = at::matmul(dy, weight.to(dy.scalar_type()));
        const int64_t O = weight.size(0), F = weight.size(1);
        Tensor rows = dy.reshape({dy.numel() / O, O});
        if (codes.defined()) {
            if (O > 1 && rows.stride(1) != 1) rows = rows.contiguous();
            dw = at::empty({O, F}, weight.options());
            if (bias && bias_type == weight.scalar_type()) db = at::empty({O}, weight.options());
            weight_grad8_launch(rows, codes, saved[2], dw, some(db));
        }
        if (bias && !db.defined()) db = rows.sum(0, false, at::kFloat).to(bias_type);
        return {dx, dw, db};
    }
};

}  // namespace

std::tuple<Tensor, Tensor> gated_scan(Tensor p, int64_t dim, c10::optional<Tensor> h0, c10::optional<Tensor> lengths, bool keep8) {
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(p) && !(h0.has_value() && dual(*h0)), "gated_scan: no forward mode (jvp)");
    if (at::GradMode::is_enabled() && (p.requires_grad() || (h0.has_value() && h0->requires_grad()))) {
        auto out = GatedScan::apply(p, h0, lengths, dim, keep8);
        return {out[0], out[1]};
    }
    Scan s = scan(p, dim, h0, lengths, false, false);
    return {s.y, s.last};
}

Tensor linear8(Tensor x, Tensor weight, c10::optional<Tensor> bias) {
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
    if (!at::GradMode::is_enabled()) return project(x, weight, bias);
    return Linear8::apply(x, weight, bias);
}
