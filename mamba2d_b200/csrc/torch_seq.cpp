// Eager entry points of the sequence operators (sequence.py): linear attention, group normalisation, clipping.
//
// Arguments are checked here (in Python the checks took longer than a small call's kernel).
#include "torch_seq.h"

void bind_layers(pybind11::module& m);            // torch_layers.cpp

namespace {

using namespace m2d_entry;

m2d_attn_tensor attn_tensor(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

// ---- linear attention -------------------------------------------------------------------------------

struct Attn {
    Tensor q, k, v, g, state, lengths;        // as the kernels read them
    m2d_attn_desc d{};
    Attn(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const Tensor& state_, const Tensor& lengths_, double scale)
        : q(rows(q_)), k(rows(k_)), v(rows(v_)), g(g_), state(dense(state_)), lengths(dense(lengths_)) {
        d.struct_bytes = sizeof(d);
        d.dtype = dtype_of(v);
        d.B = (int)v.size(0); d.T = (int)v.size(1); d.H = (int)v.size(2); d.V = (int)v.size(3);
        d.G = (int)q.size(2); d.K = (int)q.size(3);
        d.scale = (float)scale;
        d.q = attn_tensor(q); d.k = attn_tensor(k); d.v = attn_tensor(v);
        d.log_decay = fptr(g);
        const bool per_head = g.dim() == 1;
        d.g_batch = per_head ? 0 : g.stride(0);
        d.g_token = per_head ? 0 : g.stride(1);
        d.g_head = per_head ? g.stride(0) : g.stride(2);
        d.state = fptr(state);
        d.lengths = static_cast<const int32_t*>(ptr(lengths));
    }
};

Tensor attn_forward(Attn& a, Tensor* state_out) {
    const Tensor o = at::empty({a.d.B, a.d.T, a.d.H, a.d.V}, a.v.options());
    a.d.o = o.data_ptr();
    if (state_out) {
        *state_out = at::empty({a.d.B, a.d.H, a.d.K, a.d.V}, a.v.options().dtype(at::kFloat));
        a.d.state_out = fptr(*state_out);
    }
    a.d.workspace_bytes = m2d_attn_fwd_workspace(&a.d);
    Tensor ws;
    if (a.d.workspace_bytes) {
        ws = scratch(a.d.workspace_bytes, a.v);
        a.d.workspace = ws.data_ptr();
    }
    check(m2d_attn_fwd(&a.d, stream_of(a.v)), "m2d_attn_fwd");
    return o;
}

bool no_tokens(const Tensor& v) { return v.size(0) == 0 || v.size(1) == 0; }
// The state after no tokens.
Tensor same_state(const Tensor& q, const Tensor& v, const Tensor& state) {
    return state.defined() ? state.clone() : at::zeros({v.size(0), v.size(2), q.size(3), v.size(3)}, v.options().dtype(at::kFloat));
}

class AttnFn : public torch::autograd::Function<AttnFn> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const optional<Tensor>& state_,
                                 const optional<Tensor>& lengths_, double scale, bool want_state) {
        const Tensor state = or_none(state_), lengths = or_none(lengths_);
        const c10::cuda::CUDAGuard guard(v.device());
        Tensor o, out_state;
        if (no_tokens(v)) {
            o = at::empty(v.sizes(), v.options());
            if (want_state) out_state = same_state(q, v, state);
        } else {
            Attn a(q, k, v, g, state, lengths, scale);
            o = attn_forward(a, want_state ? &out_state : nullptr);
        }
        ctx->save_for_backward({q, k, v, g, state, lengths});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return want_state ? variable_list{o, out_state} : variable_list{o};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_attention: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[2].device());
        check_waits("linear_attention");
        const bool have_state_grad = grads.size() > 1 && grads[1].defined();
        if (!grads[0].defined() && !have_state_grad) return variable_list(8);
        if (no_tokens(s[2])) {
            auto none = [](const Tensor& t) { return t.defined() && t.requires_grad() ? at::zeros(t.sizes(), t.options()) : Tensor(); };
            return {none(s[0]), none(s[1]), none(s[2]), none(s[3]), have_state_grad && s[4].defined() ? grads[1] : none(s[4]), Tensor(), Tensor(), Tensor()};
        }
        Attn a(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble());
        m2d_attn_desc& d = a.d;
        const Tensor d_o = grads[0].defined() ? rows(grads[0].to(a.v.scalar_type())) : at::zeros(a.v.sizes(), a.v.options());
        const Tensor d_out = have_state_grad ? grads[1].to(at::kFloat).contiguous() : Tensor();
        d.d_o = attn_tensor(d_o);
        d.d_state_out = fptr(d_out);
        Tensor dq = at::empty({d.B, d.T, d.G, d.K}, a.v.options()), dk = at::empty_like(dq), dv = at::empty({d.B, d.T, d.H, d.V}, a.v.options());
        d.d_q = dq.data_ptr(); d.d_k = dk.data_ptr(); d.d_v = dv.data_ptr();
        Tensor dg, ds;
        if (s[3].requires_grad()) {
            dg = at::empty({d.B, d.T, d.H}, a.g.options());
            d.d_log_decay = fptr(dg);
        }
        if (s[4].defined() && s[4].requires_grad()) {
            ds = at::empty(s[4].sizes(), s[4].options());
            d.d_state = fptr(ds);
        }
        d.workspace_bytes = m2d_attn_bwd_workspace(&d);
        Tensor ws;
        if (d.workspace_bytes) {
            ws = scratch(d.workspace_bytes, a.v);
            d.workspace = ws.data_ptr();
        }
        check(m2d_attn_bwd(&d, stream_of(a.v)), "m2d_attn_bwd");
        if (dg.defined() && s[3].dim() == 1) dg = dg.sum(at::IntArrayRef{0, 1});
        return {dq, dk, dv, dg, ds, Tensor(), Tensor(), Tensor()};
    }
};

// What q, k, v, log_decay and a state have to be: (tokens..., heads, dim) with one or two dimensions of tokens.
void check_attn(const char* what, const char* tokens, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state) {
    const int64_t lead = tokens[1] ? 2 : 1;
    TORCH_CHECK(v.dim() == lead + 2, what, ": v must be (", tokens[0], lead > 1 ? ", T" : "", ", H, V), got ", v.sizes());
    TORCH_CHECK(q.dim() == v.dim() && k.sizes() == q.sizes() && q.sizes().slice(0, lead) == v.sizes().slice(0, lead), what, ": q and k must be (", tokens[0], lead > 1 ? ", T" : "",
                ", G, K) next to v ", v.sizes(), ", got ", q.sizes(), " and ", k.sizes());
    const int64_t H = v.size(lead), V = v.size(lead + 1), G = q.size(lead), K = q.size(lead + 1);
    TORCH_CHECK(H >= 1 && G >= 1 && H % G == 0, what, ": ", G, " heads of q and k cannot be shared by ", H, " heads of v");
    TORCH_CHECK(K >= 1 && K <= M2D_ATTN_MAX_DIM && V >= 1 && V <= M2D_ATTN_MAX_DIM, what, ": head sizes of 1 to ", M2D_ATTN_MAX_DIM, ", got K=", K, ", V=", V);
    TORCH_CHECK((g.dim() == 1 || g.dim() == lead + 1) && g.size(-1) == H && (g.dim() == 1 || g.sizes().slice(0, lead) == v.sizes().slice(0, lead)), what,
                ": log_decay must be one per head, or one per token and head of v ", v.sizes(), ", got ", g.sizes());
    TORCH_CHECK(g.is_floating_point(), what, ": log_decay has dtype ", g.scalar_type());
    if (state.defined())
        TORCH_CHECK(state.dim() == 4 && state.size(0) == v.size(0) && state.size(1) == H && state.size(2) == K && state.size(3) == V && state.scalar_type() == at::kFloat, what,
                    ": the state must be (B, H, K, V) = (", v.size(0), ", ", H, ", ", K, ", ", V, ") in float32, got ", state.sizes(), " ", state.scalar_type());
    for (const Tensor* t : {&q, &k, &v})
        TORCH_CHECK((t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16) && t->scalar_type() == v.scalar_type(), what, ": dtype ", t->scalar_type(),
                    "; q, k and v share one, float32 or bfloat16");
    TORCH_CHECK(v.is_cuda(), what, ": tensors must be on a CUDA device (there is no CPU path)");
    for (const Tensor* t : {&q, &k, &g, &state}) TORCH_CHECK(!t->defined() || t->device() == v.device(), what, ": tensors on ", t->device(), " and ", v.device());
    for (int64_t d = 0; d < lead; ++d) TORCH_CHECK(v.size(d) <= INT_MAX, what, ": a size out of range");
}

std::tuple<Tensor, optional<Tensor>> linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const optional<double>& scale_,
                                                      const optional<Tensor>& state_, const optional<Tensor>& lengths_, bool want_state) {
    const char* const what = "linear_attention";
    const Tensor state = or_none(state_);
    check_attn(what, "BT", q, k, v, log_decay, state);
    const Tensor lengths = token_counts(what, or_none(lengths_), v);
    if (!no_tokens(v)) check_waits(what);
    const Tensor g = log_decay.to(at::kFloat);
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)q.size(-1));
    if (wants_grad({&q, &k, &v, &g, &state})) {
        const variable_list r = AttnFn::apply(q, k, v, g, state_, lengths.defined() ? optional<Tensor>(lengths) : c10::nullopt, scale, want_state);
        return {r[0], want_state ? optional<Tensor>(r[1]) : c10::nullopt};
    }
    if (no_tokens(v)) return {v.clone(), want_state ? optional<Tensor>(same_state(q, v, state)) : c10::nullopt};
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(v.device());
    Attn a(q, k, v, g, state, lengths, scale);
    Tensor out_state;
    const Tensor o = attn_forward(a, want_state ? &out_state : nullptr);
    return {o, want_state ? optional<Tensor>(out_state) : c10::nullopt};
}

Tensor linear_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const optional<double>& scale) {
    const char* const what = "linear_attention_step";
    TORCH_CHECK(state.defined(), what, ": there is no state");
    check_attn(what, "B", q, k, v, log_decay, state);
    const int64_t B = v.size(0), H = v.size(1), K = q.size(2), V = v.size(2), span = K * V, sb = state.stride(0), sh = state.stride(1);
    const bool dense_kv = (V == 1 || state.stride(3) == 1) && (K == 1 || state.stride(2) == V);
    const bool apart = (B == 1 || sb >= span) && (H == 1 || sh >= span) && (B == 1 || H == 1 || sb >= (H - 1) * sh + span || sh >= (B - 1) * sb + span);
    TORCH_CHECK(B == 0 || (dense_kv && apart), what, ": the state must be dense in (K, V) and must not overlap itself, got strides ", state.strides());
    TORCH_CHECK(!wants_grad({&q, &k, &v, &log_decay, &state}), what, " updates the state in place and has no gradients: call it without gradients");
    if (B == 0) return v.clone();
    check_waits(what);                       // (the state may be that of a prompt)
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(v.device());
    const Tensor qr = rows(q), kr = rows(k), vr = rows(v), g = log_decay.to(at::kFloat);
    m2d_attn_desc d{};
    d.struct_bytes = sizeof(d);
    d.dtype = dtype_of(v);
    d.B = (int)B; d.T = 1; d.H = (int)H; d.V = (int)V;
    d.G = (int)q.size(1); d.K = (int)K;
    d.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)K));
    auto token = [](const Tensor& t) { return m2d_attn_tensor{t.data_ptr(), t.stride(0), 0, t.stride(1)}; };
    d.q = token(qr); d.k = token(kr); d.v = token(vr);
    d.log_decay = fptr(g);
    d.g_batch = g.dim() == 1 ? 0 : g.stride(0);
    d.g_head = g.stride(-1);
    d.state = d.state_out = fptr(state);
    const Tensor o = at::empty({d.B, d.H, d.V}, v.options());
    d.o = o.data_ptr();
    check(m2d_attn_step(&d, sb, sh, stream_of(v)), "m2d_attn_step");
    wrote(state);
    return o;
}

// ---- group normalisation ----------------------------------------------------------------------------

m2d_norm_desc norm_desc(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, int64_t act, double eps) {
    m2d_norm_desc d{};
    d.struct_bytes = sizeof(d);
    d.dtype = dtype_of(x);
    d.N = x.size(0); d.C = (int)x.size(-1);
    d.S = x.numel() / (d.N * d.C);
    d.groups = (int)groups; d.act = (int)act; d.eps = (float)eps;
    const Tensor& p = weight.defined() ? weight : bias;
    d.params_f32 = p.defined() && p.scalar_type() == at::kFloat;
    d.x = x.data_ptr(); d.weight = ptr(weight); d.bias = ptr(bias);
    return d;
}
Tensor norm_forward(m2d_norm_desc& d, const Tensor& x) {
    const Tensor y = at::empty(x.sizes(), x.options());
    d.y = y.data_ptr();
    d.workspace_bytes = m2d_norm_fwd_workspace(&d);
    Tensor ws;
    if (d.workspace_bytes) {
        ws = scratch(d.workspace_bytes, x);
        d.workspace = ws.data_ptr();
    }
    check(m2d_norm_fwd(&d, stream_of(x)), "m2d_norm_fwd");
    return y;
}

class NormFn : public torch::autograd::Function<NormFn> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const optional<Tensor>& weight_, const optional<Tensor>& bias_, int64_t groups, int64_t act, double eps) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_);
        const c10::cuda::CUDAGuard guard(x_.device());
        Tensor y, stats;
        if (x_.numel()) {
            const Tensor x = x_.contiguous(), w = dense(weight), b = dense(bias);
            m2d_norm_desc d = norm_desc(x, w, b, groups, act, eps);
            stats = at::empty({d.N, d.groups, 2}, x.options().dtype(at::kFloat));
            d.stats = fptr(stats);
            y = norm_forward(d, x);
        } else {                                   // (nothing to do, but the parameters have gradients: zero)
            y = at::empty(x_.sizes(), x_.options());
        }
        ctx->save_for_backward({x_, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["eps"] = eps;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "group_norm: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[0].device());
        if (!s[0].numel()) {
            auto none = [](const Tensor& t) { return t.defined() && t.requires_grad() ? at::zeros(t.sizes(), t.options()) : Tensor(); };
            return {at::empty(s[0].sizes(), s[0].options()), none(s[1]), none(s[2]), Tensor(), Tensor(), Tensor()};
        }
        const Tensor x = s[0].contiguous(), w = dense(s[1]), b = dense(s[2]), dy = grads[0].to(x.scalar_type()).contiguous();
        m2d_norm_desc d = norm_desc(x, w, b, ctx->saved_data["groups"].toInt(), ctx->saved_data["act"].toInt(), ctx->saved_data["eps"].toDouble());
        d.stats = fptr(s[3]);
        d.d_y = dy.data_ptr();
        const Tensor dx = at::empty(x.sizes(), x.options());
        d.d_x = dx.data_ptr();
        Tensor dw, db;
        // (asked of the inputs: a copy made here, where gradients are off, requires none)
        if ((s[1].defined() && s[1].requires_grad()) || (s[2].defined() && s[2].requires_grad())) {
            const auto options = w.defined() ? w.options() : b.options();
            dw = at::empty({d.C}, options);
            db = at::empty({d.C}, options);
            d.d_weight = dw.data_ptr();
            d.d_bias = db.data_ptr();
        }
        d.workspace_bytes = m2d_norm_bwd_workspace(&d);
        Tensor ws;
        if (d.workspace_bytes) {
            ws = scratch(d.workspace_bytes, x);
            d.workspace = ws.data_ptr();
        }
        check(m2d_norm_bwd(&d, stream_of(x)), "m2d_norm_bwd");
        return {dx, w.defined() ? dw : Tensor(), b.defined() ? db : Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor group_norm(const Tensor& x_, int64_t groups, const optional<Tensor>& weight_, const optional<Tensor>& bias_, double eps, int64_t act) {
    const Tensor weight = or_none(weight_), bias = or_none(bias_);
    TORCH_CHECK(x_.dim() >= 2, "group_norm: x must be (N, ..., C), got ", x_.sizes());
    const int64_t C = x_.size(-1);
    TORCH_CHECK_VALUE(groups >= 1 && C % groups == 0, "group_norm: ", C, " channels do not make ", groups, " groups");
    TORCH_CHECK_VALUE(eps >= 0, "group_norm: eps must not be negative, got ", eps);
    TORCH_CHECK(x_.scalar_type() == at::kFloat || x_.scalar_type() == at::kBFloat16, "group_norm: unsupported dtype ", x_.scalar_type(), " (float32 and bfloat16 only)");
    TORCH_CHECK(x_.is_cuda(), "group_norm: tensors must be on a CUDA device (there is no CPU path)");
    TORCH_CHECK(C <= INT_MAX, "group_norm: a size out of range");
    for (const Tensor* p : {&weight, &bias})
        if (p->defined()) {
            TORCH_CHECK(p->dim() == 1 && p->size(0) == C, "group_norm: weight and bias must have shape (", C, "), got ", p->sizes());
            TORCH_CHECK((p->scalar_type() == at::kFloat || p->scalar_type() == x_.scalar_type()) && (!weight.defined() || p->scalar_type() == weight.scalar_type()),
                        "group_norm: dtype ", p->scalar_type(), "; weight and bias share one, float32 or ", x_.scalar_type());
            TORCH_CHECK(p->device() == x_.device(), "group_norm: tensors on ", p->device(), " and ", x_.device());
        }
    if (wants_grad({&x_, &weight, &bias})) return NormFn::apply(x_, weight_, bias_, groups, act, eps);
    if (!x_.numel()) return x_.clone();
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(x_.device());
    const Tensor x = x_.contiguous(), w = dense(weight), b = dense(bias);
    m2d_norm_desc d = norm_desc(x, w, b, groups, act, eps);
    return norm_forward(d, x);
}

// ---- clipping ---------------------------------------------------------------------------------------

Tensor clip_grad_norm(const std::vector<Tensor>& grads, double max_norm) {
    TORCH_CHECK(!grads.empty(), "clip_norm_: no tensors");
    const Tensor& first = grads[0];
    std::vector<m2d_clip_tensor> table;
    std::vector<std::pair<const char*, const char*>> spans;
    table.reserve(grads.size());
    spans.reserve(grads.size());
    bool sorted = true;
    const bool recording = at::GradMode::is_enabled();
    for (const Tensor& g : grads) {
        TORCH_CHECK(g.is_cuda() && g.layout() == at::kStrided, "clip_norm_: tensors must be dense and on a CUDA device (there is no CPU path)");
        TORCH_CHECK(g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16, "clip_norm_: unsupported dtype ", g.scalar_type(), " (float32 and bfloat16 only)");
        TORCH_CHECK(g.device() == first.device(), "clip_norm_: tensors on ", g.device(), " and ", first.device());
        TORCH_CHECK(!recording || !g.requires_grad(), "clip_norm_: a tensor that requires a gradient is not scaled in place");
        TORCH_CHECK(g.is_contiguous() || g.is_non_overlapping_and_dense(), "clip_norm_: a tensor has gaps or overlaps itself (sizes ", g.sizes(), ", strides ", g.strides(), ")");
        const int64_t n = g.numel();
        if (!n) continue;
        const char* p = static_cast<const char*>(g.data_ptr());
        table.push_back({const_cast<char*>(p), n, dtype_of(g)});
        sorted = sorted && (spans.empty() || spans.back().second <= p);
        spans.emplace_back(p, p + n * g.element_size());
    }
    if (!sorted) {
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i) TORCH_CHECK(spans[i - 1].second <= spans[i].first, "clip_norm_: two tensors share memory");
    }
    const c10::cuda::CUDAGuard guard(first.device());
    const Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
    const uint64_t bytes = m2d_clip_workspace(table.data(), (int32_t)table.size());
    const Tensor ws = scratch(bytes, first);
    check(m2d_clip_grad_norm(table.data(), (int32_t)table.size(), (float)max_norm, fptr(norm), ws.data_ptr(), bytes, stream_of(first)), "m2d_clip_grad_norm");
    for (const Tensor& g : grads) wrote(g);
    return norm;
}

}  // namespace

void bind_sequence_operators(pybind11::module& m) {
    bind_layers(m);
    using pybind11::arg;
    m.def("linear_attention", &linear_attention, "linear attention of whole sequences: (o, state or None)", arg("q"), arg("k"), arg("v"), arg("log_decay"), arg("scale").none(true),
          arg("state").none(true), arg("lengths").none(true), arg("want_state"));
    m.def("linear_attention_step", &linear_attention_step, "linear attention of one token; the state is updated in place", arg("q"), arg("k"), arg("v"), arg("log_decay"), arg("state"),
          arg("scale").none(true));
    m.def("group_norm", &group_norm, "group normalisation with an activation, channels last", arg("x"), arg("groups"), arg("weight").none(true), arg("bias").none(true), arg("eps"), arg("act"));
    m.def("clip_grad_norm", &clip_grad_norm, "global norm; the tensors are scaled in place", arg("grads"), arg("max_norm"));
}
