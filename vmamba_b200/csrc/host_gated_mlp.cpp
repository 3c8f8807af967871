// Gated feed-forward block: argument checks, results, workspaces and the autograd node.
#include "host_common.h"

namespace host {

static ss2d_gated_mlp_params mlp_params(const Tensor& x, const Tensor& w1, const Tensor& w2, int64_t act) {
    ss2d_gated_mlp_params p = {};
    p.x = x.data_ptr(); p.w1 = w1.data_ptr(); p.w2 = w2.data_ptr();
    p.tokens = x.size(0); p.channels = x.size(1); p.hidden = w2.size(1); p.outputs = w2.size(0);
    p.x_row_stride = x.size(0) == 1 ? x.size(1) : x.stride(0);
    p.dtype = dtype_code(x); p.act = (int32_t)act;
    return p;
}
// (tokens, channels) with contiguous rows that do not overlap
static Tensor token_rows(const Tensor& x) {
    Tensor t = x.reshape({-1, x.size(-1)});
    return t.stride(1) == 1 && (t.size(0) < 2 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}

struct Fed { Tensor y, h; };
static Fed mlp_fwd(const Tensor& x, const Tensor& w1, const Tensor& w2, const Tensor& b1, const Tensor& b2, int64_t act) {
    const CallGuard guard(x);
    ss2d_gated_mlp_params p = mlp_params(x, w1, w2, act);
    Fed r;
    r.y = at::empty({p.tokens, p.outputs}, x.options());
    r.h = at::empty({p.tokens, p.hidden}, x.options());
    p.b1 = ptr(b1); p.b2 = ptr(b2); p.h = r.h.data_ptr(); p.y = r.y.data_ptr();
    const int64_t need = ss2d_gated_mlp_workspace_bytes(&p);
    Tensor ws;
    if (need > 0) { ws = bytes(need, x); p.workspace = ws.data_ptr(); p.workspace_bytes = need; }
    check(ss2d_gated_mlp_fwd(&p, stream_of(x)), "ss2d_gated_mlp_fwd");
    return r;
}

struct GatedMlpNode : public torch::autograd::Function<GatedMlpNode> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w1, const Tensor& w2, const OptT& b1, const OptT& b2, int64_t act) {
        const Fed r = mlp_fwd(x, w1, w2, opt(b1), opt(b2), act);
        ctx->save_for_backward({x, w1, w2, r.h, opt(b1)});
        ctx->saved_data["act"] = act;
        // by argument: the edges that the engine asks for are numbered without the tensors that are not there
        int64_t wanted = 0, i = 0;
        for (const Tensor& t : {x, w1, w2, opt(b1), opt(b2)}) wanted |= (int64_t)(t.defined() && t.requires_grad()) << i++;
        ctx->saved_data["wanted"] = wanted;
        return r.y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once_differentiable("gated_mlp_fn");
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w1 = s[1], &w2 = s[2];
        const CallGuard guard(x);
        const Tensor dy = token_rows(grads[0]);
        ss2d_gated_mlp_bwd_params p = {};
        p.fwd = mlp_params(x, w1, w2, ctx->saved_data["act"].toInt());
        p.fwd.h = s[3].data_ptr(); p.fwd.b1 = ptr(s[4]);
        p.dy = dy.data_ptr();
        p.dy_row_stride = dy.size(0) == 1 ? dy.size(1) : dy.stride(0);
        Tensor d[5];
        const int64_t wanted = ctx->saved_data["wanted"].toInt();
        auto want = [&](int i, at::IntArrayRef sizes) {
            if (!(wanted >> i & 1)) return (void*)nullptr;
            d[i] = at::empty(sizes, x.options());
            return d[i].data_ptr();
        };
        p.dx = want(0, x.sizes()); p.dw1 = want(1, w1.sizes()); p.dw2 = want(2, w2.sizes());
        p.db1 = want(3, {w1.size(0)}); p.db2 = want(4, {w2.size(0)});
        const int64_t need = ss2d_gated_mlp_bwd_workspace_bytes(&p);
        TORCH_CHECK(need >= 0, "ss2d_gated_mlp_bwd_workspace_bytes: invalid or unsupported arguments");
        const Tensor ws = bytes(std::max<int64_t>(need, 16), x);
        p.workspace = ws.data_ptr(); p.workspace_bytes = ws.numel();
        check(ss2d_gated_mlp_bwd(&p, stream_of(x)), "ss2d_gated_mlp_bwd");
        return {d[0], d[1], d[2], d[3], d[4], Tensor()};
    }
};

static Tensor gated_mlp_fn(const Tensor& x, const Tensor& w1, const Tensor& w2, const OptT& b1_, const OptT& b2_, int64_t act) {
    const Tensor b1 = opt(b1_), b2 = opt(b2_);
    require_on(x, {&w1, &w2, &b1, &b2});
    no_tangents("gated_mlp_fn", {&x, &w1, &w2, &b1, &b2});
    dtype_code(x);
    for (const Tensor* t : {&w1, &w2, &b1, &b2})
        TORCH_CHECK_TYPE(!t->defined() || t->scalar_type() == x.scalar_type(), "x, weights and biases must share one dtype, got ", x.scalar_type(), " and ", t->scalar_type());
    TORCH_CHECK(x.dim() >= 1 && w1.dim() == 2 && w2.dim() == 2 && w1.size(1) == x.size(-1) && w1.size(0) == 2 * w2.size(1),
                "x, w1 and w2 must be (..., channels), (2 * hidden, channels) and (outputs, hidden), got ", x.sizes(), " ", w1.sizes(), " ", w2.sizes());
    TORCH_CHECK(w1.numel() > 0 && w2.numel() > 0, "channels, hidden and outputs must not be zero");
    TORCH_CHECK(!b1.defined() || (b1.dim() == 1 && b1.size(0) == w1.size(0)), "b1 must have 2 * hidden elements");
    TORCH_CHECK(!b2.defined() || (b2.dim() == 1 && b2.size(0) == w2.size(0)), "b2 must have one element per output");
    auto shape = x.sizes().vec();
    shape.back() = w2.size(0);
    if (x.numel() == 0) {                       // no token: zeros for whoever asks for gradients
        Tensor zero = x.sum() + w1.sum() * 0 + w2.sum() * 0;
        if (b1.defined()) zero = zero + b1.sum() * 0;
        if (b2.defined()) zero = zero + b2.sum() * 0;
        return at::zeros(shape, x.options()) + zero;
    }
    auto dense = [](const Tensor& t) { return t.defined() ? OptT(t.contiguous()) : OptT(); };
    const Tensor rows = token_rows(x), v1 = w1.contiguous(), v2 = w2.contiguous();
    const OptT c1 = dense(b1), c2 = dense(b2);
    bool grad = false;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : {&x, &w1, &w2, &b1, &b2}) grad = grad || (t->defined() && t->requires_grad());
    if (grad) return GatedMlpNode::apply(rows, v1, v2, c1, c2, act).reshape(shape);
    return mlp_fwd(rows, v1, v2, opt(c1), opt(c2), act).y.view(shape);
}

void bind_gated_mlp(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("gated_mlp_fn", &gated_mlp_fn, py::call_guard<py::gil_scoped_release>());
}

}  // namespace host
