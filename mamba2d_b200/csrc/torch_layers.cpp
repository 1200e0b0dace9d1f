// Eager entry points of the gated recurrence, layer normalisation and the distillation loss (sequence.py).
#include "torch_seq.h"

namespace {

using namespace m2d_entry;

m2d_recur_tensor recur_tensor(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1)}; }

struct Recur {
    Tensor x, gate, state, lengths;           // as the kernels read them
    m2d_recur_desc d{};
    Recur(const Tensor& x_, const Tensor& gate_, const Tensor& state_, const Tensor& lengths_, int64_t form)
        : x(rows(x_)), gate(rows(gate_)), state(dense(state_)), lengths(dense(lengths_)) {
        d.struct_bytes = sizeof(d);
        d.dtype = dtype_of(x);
        d.B = (int)x.size(0); d.T = (int)x.size(1); d.C = (int)x.size(2);
        d.form = (int)form;
        d.x = recur_tensor(x); d.gate = recur_tensor(gate);
        d.lengths = static_cast<const int32_t*>(ptr(lengths));
        d.state = fptr(state);
    }
    Tensor forward(Tensor* state_out, Tensor* marks) {
        const Tensor y = at::empty({d.B, d.T, d.C}, x.options());
        d.y = y.data_ptr();
        const auto f32 = x.options().dtype(at::kFloat);
        if (state_out) {
            *state_out = at::empty({d.B, d.C}, f32);
            d.state_out = fptr(*state_out);
        }
        if (marks) {
            *marks = at::empty({(int64_t)m2d_recur_marks(&d)}, f32);
            d.marks = fptr(*marks);
        }
        check(m2d_recur_fwd(&d, stream_of(x)), "m2d_recur_fwd");
        return y;
    }
};

// The state after no tokens.
Tensor same_state(const Tensor& x, const Tensor& state) {
    return state.defined() ? state.clone() : at::zeros({x.size(0), x.size(2)}, x.options().dtype(at::kFloat));
}

class RecurFn : public torch::autograd::Function<RecurFn> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const optional<Tensor>& state_, const optional<Tensor>& lengths_, int64_t form, bool want_state) {
        const Tensor state = or_none(state_), lengths = or_none(lengths_);
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor y, state_out, marks;
        if (x.numel()) {
            Recur r(x, gate, state, lengths, form);
            y = r.forward(want_state ? &state_out : nullptr, &marks);
        } else {
            y = at::empty(x.sizes(), x.options());
            if (want_state) state_out = same_state(x, state);
        }
        ctx->save_for_backward({x, gate, state, lengths, marks});
        ctx->saved_data["form"] = form;
        ctx->set_materialize_grads(false);
        return want_state ? variable_list{y, state_out} : variable_list{y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_recurrence: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[0].device());
        check_waits("gated_recurrence");
        const bool have_state_grad = grads.size() > 1 && grads[1].defined();
        if (!grads[0].defined() && !have_state_grad) return variable_list(6);
        if (!s[0].numel()) {
            const Tensor dx = at::empty(s[0].sizes(), s[0].options());
            const Tensor ds = !s[2].defined() || !s[2].requires_grad() ? Tensor() : have_state_grad ? grads[1] : at::zeros(s[2].sizes(), s[2].options());
            return {dx, at::empty_like(dx), ds, Tensor(), Tensor(), Tensor()};
        }
        Recur r(s[0], s[1], s[2], s[3], ctx->saved_data["form"].toInt());
        m2d_recur_desc& d = r.d;
        // (no gradient of h: one zero, expanded)
        const Tensor dy = grads[0].defined() ? rows(grads[0].to(r.x.scalar_type())) : at::zeros({1, 1, d.C}, r.x.options()).expand({d.B, d.T, d.C});
        const Tensor d_out = have_state_grad ? grads[1].to(at::kFloat).contiguous() : Tensor();
        d.d_y = recur_tensor(dy);
        d.d_state_out = fptr(d_out);
        d.marks = fptr(s[4]);
        const Tensor dx = at::empty({d.B, d.T, d.C}, r.x.options()), dgate = at::empty_like(dx);
        d.d_x = dx.data_ptr();
        d.d_gate = dgate.data_ptr();
        Tensor ds;
        if (s[2].defined() && s[2].requires_grad()) {
            ds = at::empty({d.B, d.C}, s[2].options());
            d.d_state = fptr(ds);
        }
        check(m2d_recur_bwd(&d, stream_of(r.x)), "m2d_recur_bwd");
        return {dx, dgate, ds, Tensor(), Tensor(), Tensor()};
    }
};

void check_recur(const char* what, const char* shape, int64_t dims, const Tensor& x, const Tensor& gate, const Tensor& state) {
    TORCH_CHECK(x.dim() == dims && gate.sizes() == x.sizes(), what, ": x and gate must be ", shape, ", got ", x.sizes(), " and ", gate.sizes());
    for (const Tensor* t : {&x, &gate})
        TORCH_CHECK((t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16) && t->scalar_type() == x.scalar_type(), what, ": dtype ", t->scalar_type(),
                    "; x and gate share one, float32 or bfloat16");
    if (state.defined())
        TORCH_CHECK(state.dim() == 2 && state.size(0) == x.size(0) && state.size(1) == x.size(-1) && state.scalar_type() == at::kFloat, what, ": the state must be (B, C) = (", x.size(0),
                    ", ", x.size(-1), ") in float32, got ", state.sizes(), " ", state.scalar_type());
    TORCH_CHECK(x.is_cuda(), what, ": tensors must be on a CUDA device (there is no CPU path)");
    for (const Tensor* t : {&gate, &state}) TORCH_CHECK(!t->defined() || t->device() == x.device(), what, ": tensors on ", t->device(), " and ", x.device());
    for (int64_t d = 0; d < dims; ++d) TORCH_CHECK(x.size(d) <= INT_MAX, what, ": a size out of range");
}

std::tuple<Tensor, optional<Tensor>> gated_recurrence(const Tensor& x, const Tensor& gate, int64_t form, const optional<Tensor>& state_, const optional<Tensor>& lengths_, bool want_state) {
    const char* const what = "gated_recurrence";
    const Tensor state = or_none(state_);
    check_recur(what, "(B, T, C)", 3, x, gate, state);
    const Tensor lengths = token_counts(what, or_none(lengths_), x);
    const c10::cuda::CUDAGuard guard(x.device());
    if (x.numel()) check_waits(what);
    if (wants_grad({&x, &gate, &state})) {
        const variable_list r = RecurFn::apply(x, gate, state_, lengths.defined() ? optional<Tensor>(lengths) : c10::nullopt, form, want_state);
        return {r[0], want_state ? optional<Tensor>(r[1]) : c10::nullopt};
    }
    if (!x.numel()) return {x.clone(), want_state ? optional<Tensor>(same_state(x, state)) : c10::nullopt};
    const at::AutoDispatchBelowADInplaceOrView below;
    Recur r(x, gate, state, lengths, form);
    Tensor state_out;
    const Tensor y = r.forward(want_state ? &state_out : nullptr, nullptr);
    return {y, want_state ? optional<Tensor>(state_out) : c10::nullopt};
}

Tensor gated_recurrence_step(const Tensor& x, const Tensor& gate, const Tensor& state, int64_t form) {
    const char* const what = "gated_recurrence_step";
    TORCH_CHECK(state.defined(), what, ": there is no state");
    check_recur(what, "(B, C)", 2, x, gate, state);
    const int64_t B = x.size(0), C = x.size(1), sb = state.stride(0);
    TORCH_CHECK(!x.numel() || ((C == 1 || state.stride(1) == 1) && (B == 1 || sb >= C)), what, ": the state must be dense along C and must not overlap itself, got strides ", state.strides());
    TORCH_CHECK(!wants_grad({&x, &gate, &state}), what, " updates the state in place and has no gradients: call it without gradients");
    if (!x.numel()) return x.clone();
    check_waits(what);                       // (the state may be that of a prompt)
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xr = rows(x), gr = rows(gate);
    m2d_recur_desc d{};
    d.struct_bytes = sizeof(d);
    d.dtype = dtype_of(x);
    d.B = (int)B; d.T = 1; d.C = (int)C;
    d.form = (int)form;
    d.x = {xr.data_ptr(), xr.stride(0), 0};
    d.gate = {gr.data_ptr(), gr.stride(0), 0};
    d.state = d.state_out = fptr(state);
    const Tensor y = at::empty({B, C}, x.options());
    d.y = y.data_ptr();
    check(m2d_recur_step(&d, sb, stream_of(x)), "m2d_recur_step");
    wrote(state);
    return y;
}

// ---- layer normalisation ----------------------------------------------------------------------------

m2d_ln_desc ln_desc(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
    m2d_ln_desc d{};
    d.struct_bytes = sizeof(d);
    d.dtype = dtype_of(x);
    d.N = x.size(0); d.C = (int)x.size(1);
    const Tensor& p = weight.defined() ? weight : bias;
    d.params_f32 = p.defined() && p.scalar_type() == at::kFloat;
    d.eps = (float)eps;
    d.x = x.data_ptr(); d.x_row = x.stride(0);
    d.weight = ptr(weight); d.bias = ptr(bias);
    return d;
}
// As rows (N, C) with neighbours along C: a view where there is one.
Tensor matrix(const Tensor& t) {
    if (t.dim() == 2 && t.stride(1) == 1) return t;
    const Tensor m = rows(t).reshape({-1, t.size(-1)});
    return m.size(0) == 1 || m.stride(0) >= 0 ? m : m.contiguous();
}
Tensor ln_forward(m2d_ln_desc& d, const Tensor& x, const Tensor& residual, const Tensor& like, Tensor* sum) {
    Tensor r;
    if (residual.defined()) {
        r = matrix(residual);
        d.residual = r.data_ptr();
        d.residual_row = r.stride(0);
        *sum = at::empty(like.sizes(), x.options());
        d.sum = sum->data_ptr();
    }
    const Tensor y = at::empty(like.sizes(), x.options());
    d.y = y.data_ptr();
    check(m2d_ln_fwd(&d, stream_of(x)), "m2d_ln_fwd");
    return y;
}

class LnFn : public torch::autograd::Function<LnFn> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& x_, const optional<Tensor>& weight_, const optional<Tensor>& bias_, const optional<Tensor>& residual_, double eps) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_), residual = or_none(residual_);
        const c10::cuda::CUDAGuard guard(x_.device());
        Tensor y, sum, stats;
        if (x_.numel()) {
            const Tensor x = matrix(x_), w = dense(weight), b = dense(bias);
            m2d_ln_desc d = ln_desc(x, w, b, eps);
            stats = at::empty({d.N, 2}, x.options().dtype(at::kFloat));
            d.stats = fptr(stats);
            y = ln_forward(d, x, residual, x_, &sum);
        } else {                                   // (nothing to do, but the parameters have gradients: zero)
            y = at::empty(x_.sizes(), x_.options());
            if (residual.defined()) sum = at::empty(x_.sizes(), x_.options());
        }
        ctx->save_for_backward({sum.defined() ? sum : x_, weight, bias, stats});
        ctx->set_materialize_grads(false);
        return sum.defined() ? variable_list{y, sum} : variable_list{y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[0].device());
        const bool residual = grads.size() > 1;
        const Tensor ds_ = residual ? grads[1] : Tensor();
        auto none = [](const Tensor& t) { return t.defined() && t.requires_grad() ? at::zeros(t.sizes(), t.options()) : Tensor(); };
        if (!grads[0].defined()) return {ds_, none(s[1]), none(s[2]), ds_, Tensor()};          // the sum alone was used
        if (!s[0].numel()) {
            const Tensor dx = at::empty(s[0].sizes(), s[0].options());
            return {dx, none(s[1]), none(s[2]), residual ? dx : Tensor(), Tensor()};
        }
        const Tensor x = matrix(s[0]), w = dense(s[1]), b = dense(s[2]), dy = matrix(grads[0].to(x.scalar_type())), ds = ds_.defined() ? matrix(ds_.to(x.scalar_type())) : ds_;
        m2d_ln_desc d = ln_desc(x, w, b, 0.0);           // (eps is in the statistics)
        d.stats = fptr(s[3]);
        d.d_y = dy.data_ptr(); d.d_y_row = dy.stride(0);
        if (ds.defined()) { d.d_sum = ds.data_ptr(); d.d_sum_row = ds.stride(0); }
        const Tensor dx = at::empty(s[0].sizes(), x.options());
        d.d_x = dx.data_ptr();
        Tensor dw, db;
        if (s[1].defined() && s[1].requires_grad()) { dw = at::empty({d.C}, s[1].options()); d.d_weight = dw.data_ptr(); }
        if (s[2].defined() && s[2].requires_grad()) { db = at::empty({d.C}, s[2].options()); d.d_bias = db.data_ptr(); }
        d.workspace_bytes = m2d_ln_bwd_workspace(&d);
        Tensor ws;
        if (d.workspace_bytes) {
            ws = scratch(d.workspace_bytes, x);
            d.workspace = ws.data_ptr();
        }
        check(m2d_ln_bwd(&d, stream_of(x)), "m2d_ln_bwd");
        return {dx, dw, db, residual ? dx : Tensor(), Tensor()};
    }
};

std::tuple<Tensor, optional<Tensor>> layer_norm(const Tensor& x_, const optional<Tensor>& weight_, const optional<Tensor>& bias_, const optional<Tensor>& residual_, double eps) {
    const Tensor weight = or_none(weight_), bias = or_none(bias_), residual = or_none(residual_);
    TORCH_CHECK(x_.dim() >= 1, "layer_norm: x must be (..., C), got a single value");
    const int64_t C = x_.size(-1);
    TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative, got ", eps);
    TORCH_CHECK(x_.scalar_type() == at::kFloat || x_.scalar_type() == at::kBFloat16, "layer_norm: unsupported dtype ", x_.scalar_type(), " (float32 and bfloat16 only)");
    for (const Tensor* p : {&weight, &bias})
        if (p->defined()) {
            TORCH_CHECK(p->dim() == 1 && p->size(0) == C, "layer_norm: weight and bias must have shape (", C, "), got ", p->sizes());
            TORCH_CHECK((p->scalar_type() == at::kFloat || p->scalar_type() == x_.scalar_type()) && (!weight.defined() || p->scalar_type() == weight.scalar_type()),
                        "layer_norm: dtype ", p->scalar_type(), "; weight and bias share one, float32 or ", x_.scalar_type());
        }
    if (residual.defined())
        TORCH_CHECK(residual.sizes() == x_.sizes() && residual.scalar_type() == x_.scalar_type(), "layer_norm: the residual must be like x ", x_.sizes(), " ", x_.scalar_type(), ", got ",
                    residual.sizes(), " ", residual.scalar_type());
    TORCH_CHECK(x_.is_cuda(), "layer_norm: tensors must be on a CUDA device (there is no CPU path)");
    for (const Tensor* p : {&weight, &bias, &residual}) TORCH_CHECK(!p->defined() || p->device() == x_.device(), "layer_norm: tensors on ", p->device(), " and ", x_.device());
    TORCH_CHECK(C <= INT_MAX && x_.numel() / std::max<int64_t>(C, 1) <= INT_MAX, "layer_norm: a size out of range");
    const c10::cuda::CUDAGuard guard(x_.device());
    if (wants_grad({&x_, &weight, &bias, &residual})) {
        const variable_list r = LnFn::apply(x_, weight_, bias_, residual_, eps);
        return {r[0], r.size() > 1 ? optional<Tensor>(r[1]) : c10::nullopt};
    }
    if (!x_.numel()) return {x_.clone(), residual.defined() ? optional<Tensor>(x_ + residual) : c10::nullopt};
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = matrix(x_), w = dense(weight), b = dense(bias);
    m2d_ln_desc d = ln_desc(x, w, b, eps);
    Tensor sum;
    const Tensor y = ln_forward(d, x, residual, x_, &sum);
    return {y, sum.defined() ? optional<Tensor>(sum) : c10::nullopt};
}

// ---- distillation -----------------------------------------------------------------------------------

struct Distill {
    Tensor z, t, index, labels;               // as the kernels read them: rows
    m2d_distill_desc d{};
    Distill(const Tensor& z_, const Tensor& t_, const Tensor& index_, const Tensor& labels_, double temperature, double weight)
        : z(matrix(z_)), t(matrix(t_)), index(matrix(index_)), labels(labels_.defined() ? labels_.reshape(-1).contiguous() : labels_) {
        d.struct_bytes = sizeof(d);
        d.dtype = dtype_of(z);
        d.teacher_dtype = dtype_of(t);
        d.N = z.size(0); d.V = (int)z.size(1); d.K = (int)t.size(1);
        d.index_64 = index.scalar_type() == at::kLong;
        d.labels_64 = labels.defined() && labels.scalar_type() == at::kLong;
        d.temperature = (float)temperature;
        d.label_weight = (float)weight;
        d.logits = z.data_ptr(); d.logits_row = z.stride(0);
        d.teacher = t.data_ptr(); d.teacher_row = t.stride(0);
        d.index = index.data_ptr(); d.index_row = index.stride(0);
        d.labels = ptr(labels);
    }
    Tensor forward(at::IntArrayRef shape, Tensor* stats) {
        const auto f32 = z.options().dtype(at::kFloat);
        const Tensor loss = at::empty(shape, f32);
        d.loss = fptr(loss);
        if (stats) {
            *stats = at::empty({(int64_t)m2d_distill_stats(&d)}, f32);
            d.stats = fptr(*stats);
        }
        d.workspace_bytes = m2d_distill_fwd_workspace(&d);
        Tensor ws;
        if (d.workspace_bytes) {
            ws = scratch(d.workspace_bytes, z);
            d.workspace = ws.data_ptr();
        }
        check(m2d_distill_fwd(&d, stream_of(z)), "m2d_distill_fwd");
        return loss;
    }
};

class DistillFn : public torch::autograd::Function<DistillFn> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& t, const Tensor& index, const optional<Tensor>& labels_, double temperature, double weight) {
        const Tensor labels = or_none(labels_);
        const c10::cuda::CUDAGuard guard(z.device());
        Distill r(z, t, index, labels, temperature, weight);
        Tensor stats;
        const Tensor loss = r.forward(z.sizes().slice(0, z.dim() - 1), &stats);
        ctx->save_for_backward({z, t, index, labels, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["weight"] = weight;
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "distillation_loss: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[0].device());
        Distill r(s[0], s[1], s[2], s[3], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["weight"].toDouble());
        const Tensor up = grads[0].to(at::kFloat).reshape(-1);
        r.d.d_loss = fptr(up);
        r.d.d_loss_row = up.size(0) > 1 ? up.stride(0) : 0;
        r.d.stats = fptr(s[4]);
        const Tensor dz = at::empty(s[0].sizes(), r.z.options());
        r.d.d_logits = dz.data_ptr();
        check(m2d_distill_bwd(&r.d, stream_of(r.z)), "m2d_distill_bwd");
        return {dz, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor distillation_loss(const Tensor& z, const Tensor& t, const Tensor& index, const optional<Tensor>& labels_, double temperature, double weight) {
    const char* const what = "distillation_loss";
    const Tensor labels = or_none(labels_);
    auto whole = [](const Tensor& i) { return i.scalar_type() == at::kInt || i.scalar_type() == at::kLong; };
    auto real = [](const Tensor& f) { return f.scalar_type() == at::kFloat || f.scalar_type() == at::kBFloat16; };
    TORCH_CHECK(z.dim() >= 1 && t.dim() == z.dim() && index.sizes() == t.sizes() && t.sizes().slice(0, t.dim() - 1) == z.sizes().slice(0, z.dim() - 1), what,
                ": logits (..., V) and the teacher's logits and indices (..., K) do not match, got ", z.sizes(), ", ", t.sizes(), " and ", index.sizes());
    TORCH_CHECK(t.size(-1) >= 1 && t.size(-1) <= M2D_DISTILL_MAX_TOP && z.size(-1) >= 1, what, ": 1 to ", M2D_DISTILL_MAX_TOP, " logits of the teacher and at least one class, got ", t.sizes(),
                " and ", z.sizes());
    TORCH_CHECK(z.size(-1) <= INT_MAX, what, ": a size out of range");
    TORCH_CHECK(real(z) && real(t), what, ": dtype ", z.scalar_type(), " and ", t.scalar_type(), " (float32 and bfloat16 only)");
    TORCH_CHECK(whole(index), what, ": indices must be integers, got ", index.scalar_type());
    TORCH_CHECK_VALUE(temperature > 0 && (float)temperature > 0.f && std::isfinite((float)temperature), what, ": the temperature must be positive, got ", temperature);
    TORCH_CHECK_VALUE(weight >= 0 && weight <= 1, what, ": label_weight must be in 0 ... 1, got ", weight);
    TORCH_CHECK_VALUE(labels.defined() == (weight > 0), what, ": labels and a label_weight above 0 go together");
    if (labels.defined())
        TORCH_CHECK(whole(labels) && labels.sizes() == z.sizes().slice(0, z.dim() - 1), what, ": labels must be one integer a row of ", z.sizes(), ", got ", labels.sizes(), " ",
                    labels.scalar_type());
    TORCH_CHECK(z.is_cuda(), what, ": tensors must be on a CUDA device (there is no CPU path)");
    for (const Tensor* p : std::initializer_list<const Tensor*>{&t, &index, &labels}) TORCH_CHECK(!p->defined() || p->device() == z.device(), what, ": tensors on ", p->device(), " and ", z.device());
    TORCH_CHECK(!wants_grad({&t}), what, ": the teacher gets no gradient: detach its logits");
    const c10::cuda::CUDAGuard guard(z.device());
    if (!z.numel()) return z.sum(-1).to(at::kFloat);
    if (wants_grad({&z})) return DistillFn::apply(z, t, index, labels.defined() ? optional<Tensor>(labels) : c10::nullopt, temperature, weight);
    const at::AutoDispatchBelowADInplaceOrView below;
    Distill r(z, t, index, labels, temperature, weight);
    return r.forward(z.sizes().slice(0, z.dim() - 1), nullptr);
}

}  // namespace

void bind_layers(pybind11::module& m) {
    using pybind11::arg;
    m.def("gated_recurrence", &gated_recurrence, "gated recurrence of whole sequences: (h, state or None)", arg("x"), arg("gate"), arg("form"), arg("state").none(true), arg("lengths").none(true),
          arg("want_state"));
    m.def("gated_recurrence_step", &gated_recurrence_step, "gated recurrence of one token; the state is updated in place", arg("x"), arg("gate"), arg("state"), arg("form"));
    m.def("layer_norm", &layer_norm, "layer normalisation of rows: (y, the sum that was normalised or None)", arg("x"), arg("weight").none(true), arg("bias").none(true),
          arg("residual").none(true), arg("eps"));
    m.def("distillation_loss", &distillation_loss, "distillation from a teacher's top logits, a loss a row", arg("logits"), arg("teacher"), arg("index"), arg("labels").none(true),
          arg("temperature"), arg("label_weight"));
}
