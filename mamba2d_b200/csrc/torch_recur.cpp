// Eager entry points of the gated recurrence (sequence.py).
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

class RecurFn : public torch::autograd::Function<RecurFn> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const optional<Tensor>& state_, const optional<Tensor>& lengths_, int64_t form, bool want_state) {
        const Tensor state = or_none(state_), lengths = or_none(lengths_);
        const c10::cuda::CUDAGuard guard(x.device());
        Recur r(x, gate, state, lengths, form);
        Tensor state_out, marks;
        const Tensor y = r.forward(want_state ? &state_out : nullptr, &marks);
        ctx->save_for_backward({x, gate, state, lengths, marks});
        ctx->saved_data["form"] = form;
        ctx->set_materialize_grads(false);
        return want_state ? variable_list{y, state_out} : variable_list{y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_recurrence: gradients of gradients (create_graph) are not supported");
        const variable_list s = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard guard(s[0].device());
        const bool have_state_grad = grads.size() > 1 && grads[1].defined();
        if (!grads[0].defined() && !have_state_grad) return variable_list(6);
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
    if (!x.numel()) {
        if (!want_state) return {x.clone(), c10::nullopt};
        return {x.clone(), state.defined() ? state.clone() : at::zeros({x.size(0), x.size(2)}, x.options().dtype(at::kFloat))};
    }
    if (wants_grad({&x, &gate, &state})) {
        const variable_list r = RecurFn::apply(x, gate, state_, lengths.defined() ? optional<Tensor>(lengths) : c10::nullopt, form, want_state);
        return {r[0], want_state ? optional<Tensor>(r[1]) : c10::nullopt};
    }
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

}  // namespace

void bind_recurrence(pybind11::module& m) {
    using pybind11::arg;
    m.def("gated_recurrence", &gated_recurrence, "gated recurrence of whole sequences: (h, state or None)", arg("x"), arg("gate"), arg("form"), arg("state").none(true), arg("lengths").none(true),
          arg("want_state"));
    m.def("gated_recurrence_step", &gated_recurrence_step, "gated recurrence of one token; the state is updated in place", arg("x"), arg("gate"), arg("state"), arg("form"));
}
