// Linear attention with a decay for each head: argument checks, results, workspaces and the autograd node.
#include "host_common.h"

namespace host {

static bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// of a dimension of one element any stride will do; 0 keeps rows aligned
static int64_t stride_of(const Tensor& t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

static ss2d_linear_attention_params attention_params(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double scale) {
    ss2d_linear_attention_params p = {};
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.log_decay = g.data_ptr();
    p.batch = v.size(0); p.seqlen = v.size(1); p.n_groups = q.size(2); p.heads = v.size(2); p.dk = q.size(3); p.dv = v.size(3);
    p.q_batch_stride = stride_of(q, 0); p.q_token_stride = stride_of(q, 1); p.q_head_stride = stride_of(q, 2);
    p.k_batch_stride = stride_of(k, 0); p.k_token_stride = stride_of(k, 1); p.k_head_stride = stride_of(k, 2);
    p.v_batch_stride = stride_of(v, 0); p.v_token_stride = stride_of(v, 1); p.v_head_stride = stride_of(v, 2);
    p.decay_batch_stride = g.stride(0); p.decay_token_stride = g.stride(1); p.decay_head_stride = g.stride(2);
    p.dtype = dtype_code(v);
    p.scale = (float)scale;
    return p;
}

struct Attended { Tensor out, state, chunk_states; };

// q, k, v with contiguous rows, log_decay fp32 (B, L, H), initial state fp32 or undefined
static Attended attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& s0, double scale, bool final_state, bool train) {
    const CallGuard guard(v);
    ss2d_linear_attention_params p = attention_params(q, k, v, g, scale);
    const auto f32o = v.options().dtype(at::kFloat);
    Attended r;
    r.out = at::empty(v.sizes(), v.options());
    p.out = r.out.data_ptr();
    p.initial_state = ptr(s0);
    if (final_state) { r.state = at::empty({p.batch, p.heads, p.dk, p.dv}, f32o); p.final_state = r.state.data_ptr(); }
    if (train) { r.chunk_states = bytes(std::max<int64_t>(ss2d_linear_attention_states_bytes(&p), 16), v); p.chunk_states = r.chunk_states.data_ptr(); }
    const int64_t need = ss2d_linear_attention_workspace_bytes(&p);
    Tensor ws;
    if (need > 0) { ws = bytes(need, v); p.workspace = ws.data_ptr(); p.workspace_bytes = need; }
    check(ss2d_linear_attention_fwd(&p, stream_of(v)), "ss2d_linear_attention_fwd");
    return r;
}

struct AttentionNode : public torch::autograd::Function<AttentionNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                                  const OptT& start, double scale, bool final_state) {
        const Tensor s0 = opt(start);
        const Attended r = attention_fwd(q, k, v, g, s0, scale, final_state, true);
        ctx->save_for_backward({q, k, v, g, r.chunk_states});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["start"] = s0.defined();
        ctx->set_materialize_grads(false);
        if (!final_state) return {r.out};
        return {r.out, r.state};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once_differentiable("linear_attention_fn");
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &g = s[3];
        const bool start = ctx->saved_data["start"].toBool();
        if (!grads[0].defined() && !(grads.size() > 1 && grads[1].defined())) return torch::autograd::variable_list(7);
        const CallGuard guard(v);
        const Tensor dout = grads[0].defined() ? rows(grads[0]) : at::zeros(v.sizes(), v.options());
        const Tensor dlast = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
        ss2d_linear_attention_bwd_params p = {};
        p.fwd = attention_params(q, k, v, g, ctx->saved_data["scale"].toDouble());
        p.fwd.chunk_states = s[4].data_ptr();
        p.dout = dout.data_ptr(); p.dfinal_state = ptr(dlast);
        p.dout_batch_stride = stride_of(dout, 0); p.dout_token_stride = stride_of(dout, 1); p.dout_head_stride = stride_of(dout, 2);
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        Tensor dg = at::empty(g.sizes(), g.options()), ds;
        p.dq = dq.data_ptr(); p.dk = dk.data_ptr(); p.dv = dv.data_ptr(); p.dlog_decay = dg.data_ptr();
        if (start) { ds = at::empty({p.fwd.batch, p.fwd.heads, p.fwd.dk, p.fwd.dv}, g.options()); p.dinitial_state = ds.data_ptr(); }
        const int64_t need = ss2d_linear_attention_bwd_workspace_bytes(&p);
        TORCH_CHECK(need >= 0, "ss2d_linear_attention_bwd_workspace_bytes: invalid or unsupported arguments");
        const Tensor ws = bytes(std::max<int64_t>(need, 16), v);
        p.workspace = ws.data_ptr(); p.workspace_bytes = ws.numel();
        check(ss2d_linear_attention_bwd(&p, stream_of(v)), "ss2d_linear_attention_bwd");
        return {dq, dk, dv, dg, ds, Tensor(), Tensor()};
    }
};

static void check_types(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& s0) {
    require_on(v, {&q, &k, &g, &s0});
    dtype_code(v);
    TORCH_CHECK_TYPE(q.scalar_type() == v.scalar_type() && k.scalar_type() == v.scalar_type(), "q, k and v must share one dtype");
    TORCH_CHECK_TYPE(at::isFloatingType(g.scalar_type()), "log_decay must be a floating-point tensor");
}

static std::pair<Tensor, OptT> attention_fn(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay, std::optional<double> scale_,
                                            const OptT& state_, bool final_state) {
    const Tensor state = opt(state_);
    check_types(q_, k_, v_, decay, state);
    no_tangents("linear_attention_fn", {&q_, &k_, &v_, &decay, &state});
    TORCH_CHECK(q_.dim() == 4 && v_.dim() == 4 && k_.sizes() == q_.sizes() && q_.size(0) == v_.size(0) && q_.size(1) == v_.size(1),
                "q and k must be (batch, tokens, groups, dk) and v (batch, tokens, heads, dv), got ", q_.sizes(), " ", k_.sizes(), " ", v_.sizes());
    const int64_t B = v_.size(0), L = v_.size(1), G = q_.size(2), H = v_.size(2), dk = q_.size(3), dv = v_.size(3);
    TORCH_CHECK(G > 0 && H > 0 && H % G == 0, "heads must be a multiple of the groups that q and k have, got ", H, " and ", G);
    TORCH_CHECK(dk > 0 && dv > 0, "dk and dv must not be zero");
    TORCH_CHECK((decay.dim() == 3 && decay.size(0) == B && decay.size(1) == L && decay.size(2) == H) || (decay.dim() == 1 && decay.size(0) == H),
                "log_decay must be (batch, tokens, heads) or (heads,), got ", decay.sizes());
    TORCH_CHECK(!state.defined() || (state.dim() == 4 && state.size(0) == B && state.size(1) == H && state.size(2) == dk && state.size(3) == dv),
                "initial_state must be (batch, heads, dk, dv)");
    TORCH_CHECK(!state.defined() || at::isFloatingType(state.scalar_type()), "initial_state must be a floating-point tensor");
    const double scale = scale_.value_or(1.0 / std::sqrt((double)dk));
    const Tensor s0 = state.defined() ? state.to(at::kFloat).contiguous() : Tensor();
    if (B == 0 || L == 0) {                     // no token: nothing but the state, and zeros for whoever asks for gradients
        Tensor none = v_ + (q_.sum() + k_.sum() + decay.sum().to(v_.scalar_type())) * 0;
        if (s0.defined()) none = none + s0.sum().to(v_.scalar_type()) * 0;
        if (!final_state) return {none, OptT()};
        return {none, s0.defined() ? s0.clone() : at::zeros({B, H, dk, dv}, v_.options().dtype(at::kFloat))};
    }
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
    const Tensor g = decay.to(at::kFloat).expand({B, L, H});
    if (!wants_grad({&q, &k, &v, &g, &s0})) {
        const Attended r = attention_fwd(q, k, v, g, s0, scale, final_state, false);
        return {r.out, final_state ? OptT(r.state) : OptT()};
    }
    auto r = AttentionNode::apply(q, k, v, g, s0.defined() ? OptT(s0) : OptT(), scale, final_state);
    return {r[0], final_state ? OptT(r[1]) : OptT()};
}

// Two sets of states of `size` elements, each set evenly spaced: whether any of one touches any of the other.  Both are walked in the order of their addresses.
static bool states_overlap(const Tensor& x, const Tensor& y, int64_t size) {
    const int64_t n = x.size(0), sx = x.stride(0), sy = y.stride(0), ahead = y.data_ptr<float>() - x.data_ptr<float>();
    for (int64_t i = 0, j = 0; i < n && j < n;) {
        const int64_t d = j * sy + ahead - i * sx;              // from the one to the other
        if (d > -size && d < size) return true;
        d > 0 ? ++i : ++j;
    }
    return false;
}

static std::pair<Tensor, Tensor> attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay, const Tensor& state,
                                                std::optional<double> scale_, const OptT& out_) {
    Tensor to = opt(out_);
    check_types(q_, k_, v_, decay, state);
    require_on(v_, {&to});
    no_tangents("linear_attention_step", {&q_, &k_, &v_, &decay, &state, &to});
    TORCH_CHECK(!wants_grad({&q_, &k_, &v_, &decay, &state, &to}),
                "linear_attention_step has no backward pass: call it under torch.no_grad(), or linear_attention_fn for training");
    TORCH_CHECK(q_.dim() == 3 && v_.dim() == 3 && k_.sizes() == q_.sizes() && q_.size(0) == v_.size(0),
                "q and k must be (batch, groups, dk) and v (batch, heads, dv), got ", q_.sizes(), " ", k_.sizes(), " ", v_.sizes());
    const int64_t B = v_.size(0), G = q_.size(1), H = v_.size(1), dk = q_.size(2), dv = v_.size(2);
    TORCH_CHECK(G > 0 && H > 0 && H % G == 0, "heads must be a multiple of the groups that q and k have, got ", H, " and ", G);
    TORCH_CHECK(dk > 0 && dv > 0, "dk and dv must not be zero");
    TORCH_CHECK((decay.dim() == 2 && decay.size(0) == B && decay.size(1) == H) || (decay.dim() == 1 && decay.size(0) == H),
                "log_decay must be (batch, heads) or (heads,), got ", decay.sizes());
    const int64_t size = H * dk * dv;
    auto check_state = [&](const Tensor& s, const char* name) {
        TORCH_CHECK_TYPE(s.scalar_type() == at::kFloat, name, " must be float32, got ", s.scalar_type());
        TORCH_CHECK(s.dim() == 4 && s.size(0) == B && s.size(1) == H && s.size(2) == dk && s.size(3) == dv, name, " must be (batch, heads, dk, dv)");
        TORCH_CHECK(B == 0 || (s[0].is_contiguous() && (B == 1 || s.stride(0) >= size)), name, " must be dense but for its batch stride");
    };
    check_state(state, "state");
    if (to.defined()) {
        check_state(to, "state_out");
        TORCH_CHECK(B == 0 || (state.data_ptr() == to.data_ptr() && (B == 1 || state.stride(0) == to.stride(0))) || !states_overlap(state, to, size),
                    "state_out must be state itself or memory that does not overlap it");
    } else
        to = at::empty({B, H, dk, dv}, state.options());
    const Tensor o = at::empty({B, H, dv}, v_.options());
    if (B == 0) return {o, to};
    const CallGuard guard(v_);
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_), g = decay.to(at::kFloat).expand({B, H});
    ss2d_linear_attention_step_params p = {};
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.log_decay = g.data_ptr();
    p.state = state.data_ptr(); p.state_out = to.data_ptr(); p.out = o.data_ptr();
    p.batch = B; p.n_groups = G; p.heads = H; p.dk = dk; p.dv = dv;
    p.q_batch_stride = q.stride(0); p.q_head_stride = q.stride(1); p.k_batch_stride = k.stride(0); p.k_head_stride = k.stride(1);
    p.v_batch_stride = v.stride(0); p.v_head_stride = v.stride(1); p.decay_batch_stride = g.stride(0); p.decay_head_stride = g.stride(1);
    p.state_batch_stride = B == 1 ? size : state.stride(0); p.state_out_batch_stride = B == 1 ? size : to.stride(0);
    p.dtype = dtype_code(v);
    p.scale = (float)scale_.value_or(1.0 / std::sqrt((double)dk));
    check(ss2d_linear_attention_step(&p, stream_of(v)), "ss2d_linear_attention_step");
    if (!to.is_inference()) to.unsafeGetTensorImpl()->bump_version();       // a graph that has kept what was there is told
    return {o, to};
}

void bind_attention(pybind11::module_& m) {
    namespace py = pybind11;
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("linear_attention_fn", &attention_fn, release());
    m.def("linear_attention_step", &attention_step, release());
}

}  // namespace host
