// torch binding of the gated delta rule (include/rwkv7m_gated_delta.h):
// argument checks, outputs and workspaces from torch's allocator, the current
// stream, and the autograd node.  Host code only; part of _lm_head_torch.so.

#include "../../include/rwkv7m_gated_delta.h"
#include "torch_common.h"

namespace {

// The inputs as the kernels take them, copied only where they do not lie as
// needed.
struct Inputs {
    rwkv7m_gated_delta_inputs in{};
    Tensor q, k, v, g, beta;

    // strides of batch, token and head (0 along an axis of one)
    static void strides(const Tensor& t, int64_t (&to)[3]) {
        for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : 0;
    }
    // `t` where it lies, if its last axis is dense and every row starts at a
    // multiple of `align` bytes, else a copy.
    static Tensor rows(const Tensor& t, int64_t align) {
        const int64_t unit = t.element_size();
        bool fits = t.stride(3) == 1 &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % align == 0;
        for (int i = 0; i < 3; ++i)
            fits = fits && (t.size(i) <= 1 || t.stride(i) * unit % align == 0);
        // (a dense tensor that starts elsewhere is its own contiguous())
        return fits ? t : t.clone(at::MemoryFormat::Contiguous);
    }

    static void gate_shape(const char* what, const Tensor& t, int64_t B,
                           int64_t T, int64_t Hv) {
        TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == B && t.size(1) == T &&
                              t.size(2) == Hv,
                          what, " must have shape (", B, ", ", T, ", ", Hv,
                          "), got ", shape_of(t.sizes()));
    }

    Inputs(const Tensor& q_, const Tensor& k_, const Tensor& v_,
           const Tensor& g_, const Tensor& beta_, std::optional<double> scale) {
        in.dtype = code_of("q", q_);
        TORCH_CHECK_TYPE(k_.scalar_type() == q_.scalar_type() &&
                             v_.scalar_type() == q_.scalar_type(),
                         "q, k and v must share one dtype, got ",
                         q_.scalar_type(), ", ", k_.scalar_type(), " and ",
                         v_.scalar_type());
        in.g_dtype = code_of("g", g_);
        in.beta_dtype = code_of("beta", beta_);
        TORCH_CHECK_VALUE(q_.dim() == 4, "q must have shape (batch, time, "
                          "heads, head_size), got ", shape_of(q_.sizes()));
        TORCH_CHECK_VALUE(k_.sizes() == q_.sizes(), "k must have shape ",
                          shape_of(q_.sizes()), ", got ",
                          shape_of(k_.sizes()));
        in.B = q_.size(0);
        in.T = q_.size(1);
        in.Hk = q_.size(2);
        in.Dk = q_.size(3);
        TORCH_CHECK_VALUE(v_.dim() == 4 && v_.size(0) == in.B &&
                              v_.size(1) == in.T,
                          "v must have shape (", in.B, ", ", in.T,
                          ", heads, head_size), got ", shape_of(v_.sizes()));
        in.Hv = v_.size(2);
        in.Dv = v_.size(3);
        TORCH_CHECK_VALUE(in.Hk >= 1 && in.Hv >= 1 && in.Hv % in.Hk == 0,
                          "v's heads (", in.Hv, ") must be a multiple of q's "
                          "and k's (", in.Hk, ")");
        TORCH_CHECK_VALUE(in.Dk >= 8 && in.Dk <= 128 && in.Dk % 8 == 0 &&
                              in.Dv >= 8 && in.Dv <= 256 && in.Dv % 8 == 0,
                          "head sizes must be multiples of 8, q's and k's up "
                          "to 128, v's up to 256; got ", in.Dk, " and ",
                          in.Dv);
        gate_shape("g", g_, in.B, in.T, in.Hv);
        gate_shape("beta", beta_, in.B, in.T, in.Hv);
        in.scale = scale ? *scale : 1.0 / std::sqrt(double(in.Dk));
        q = q_;
        k = k_;
        v = v_;
        g = g_;
        beta = beta_;
    }
    // (on the device of the tensors, which a copy may need)
    void place() {
        if (in.B == 0 || in.T == 0) return;
        q = rows(q, 16);
        k = rows(k, 16);
        v = rows(v, 16);
        in.q = q.data_ptr();
        in.k = k.data_ptr();
        in.v = v.data_ptr();
        in.g = g.data_ptr();
        in.beta = beta.data_ptr();
        strides(q, in.q_stride);
        strides(k, in.k_stride);
        strides(v, in.v_stride);
        strides(g, in.g_stride);
        strides(beta, in.beta_stride);
    }
    std::vector<int64_t> o_shape() const {
        return {in.B, in.T, in.Hv, in.Dv};
    }
    std::vector<int64_t> state_shape() const {
        return {in.B, in.Hv, in.Dv, in.Dk};
    }
};

Tensor workspace(const Tensor& like, int64_t bytes) {
    return at::empty({bytes > 0 ? bytes : 1},
                     like.options().dtype(at::kByte).requires_grad(false));
}

// A state as the kernels take it.
Tensor placed(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

void check_state(const Inputs& x, const Tensor& initial) {
    same_gpu({&x.q, &x.k, &x.v, &x.g, &x.beta, &initial});
    if (!initial.defined()) return;
    TORCH_CHECK_VALUE(initial.sizes() == at::IntArrayRef(x.state_shape()),
                      "initial_state must have shape ",
                      shape_of(x.state_shape()), ", got ",
                      shape_of(initial.sizes()));
    TORCH_CHECK_TYPE(initial.scalar_type() == at::kFloat,
                     "initial_state must be float32, got ",
                     initial.scalar_type());
}

// [o, final state, what the backward takes (undefined where not wanted)]
variable_list rule_forward(Inputs& x, const Tensor& initial, bool train) {
    check_state(x, initial);
    const c10::DeviceGuard guard(x.q.device());
    x.place();
    const Tensor s0 = placed(initial);
    Tensor o = at::empty(x.o_shape(), x.q.options().requires_grad(false));
    Tensor end = at::empty(x.state_shape(), f32(x.q)), saved;
    if (train) {
        const int64_t n = rwkv7m_gated_delta_saved_floats(&x.in);
        saved = at::empty({n > 0 ? n : 1}, f32(x.q));
    }
    const int64_t bytes =
        train ? 0 : rwkv7m_gated_delta_workspace_bytes(&x.in, 0);
    const Tensor ws = workspace(x.q, bytes);
    check("rwkv7m_gated_delta_rule",
          rwkv7m_gated_delta_rule(&x.in, ptr<float>(s0), ptr(o),
                                  ptr<float>(end), ptr<float>(saved), ptr(ws),
                                  bytes, stream_of(x.q)));
    return {o, end, saved};
}

struct GatedDeltaRule : torch::autograd::Function<GatedDeltaRule> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q,
                                 const Tensor& k, const Tensor& v,
                                 const Tensor& g, const Tensor& beta,
                                 const OptTensor& initial,
                                 std::optional<double> scale) {
        Inputs x(q, k, v, g, beta, scale);
        const Tensor s0 = or_undefined(initial);
        auto out = rule_forward(x, s0, true);
        ctx->save_for_backward({q, k, v, g, beta, out[2]});
        ctx->saved_data["scale"] = x.in.scale;
        ctx->saved_data["state"] = s0.defined();
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        variable_list none(7);
        if (!d[0].defined() && !d[1].defined()) return none;
        no_tangents("gated_delta_rule", {&d[0], &d[1]});
        const auto s = ctx->get_saved_variables();
        Inputs x(s[0], s[1], s[2], s[3], s[4],
                 ctx->saved_data["scale"].toDouble());
        const c10::DeviceGuard guard(x.q.device());
        x.place();
        Tensor dout = d[0];
        if (!dout.defined())
            dout = at::zeros(x.o_shape(), x.q.options().requires_grad(false));
        dout = Inputs::rows(dout, 16);
        const Tensor dend = placed(d[1]);
        const auto like = [](const Tensor& t) {
            return at::empty(t.sizes(), t.options().requires_grad(false));
        };
        Tensor dq = like(s[0]), dk = like(s[1]), dv = like(s[2]),
               dg = like(s[3]), db = like(s[4]), ds0;
        if (ctx->saved_data["state"].toBool() && ctx->needs_input_grad(5))
            ds0 = at::empty(x.state_shape(), f32(x.q));
        const int64_t bytes = rwkv7m_gated_delta_workspace_bytes(&x.in, 1);
        const Tensor ws = workspace(x.q, bytes);
        int64_t stride[3];
        Inputs::strides(dout, stride);
        check("rwkv7m_gated_delta_rule_backward",
              rwkv7m_gated_delta_rule_backward(
                  &x.in, ptr(dout), stride, ptr<float>(dend),
                  ptr<float>(s[5]), ptr(dq), ptr(dk), ptr(dv), ptr(dg),
                  ptr(db), ptr<float>(ds0), ptr(ws), bytes, stream_of(x.q)));
        return once("gated_delta_rule",
                    {dq, dk, dv, dg, db, ds0, Tensor()});
    }
};

std::tuple<Tensor, Tensor> gated_delta_rule(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
    const Tensor& beta, const OptTensor& initial,
    std::optional<double> scale) {
    const Tensor s0 = or_undefined(initial);
    no_tangents("gated_delta_rule", {&q, &k, &v, &g, &beta, &s0});
    if (wants_grad({&q, &k, &v, &g, &beta, &s0})) {
        const auto out =
            GatedDeltaRule::apply(q, k, v, g, beta, initial, scale);
        return {out[0], out[1]};
    }
    Inputs x(q, k, v, g, beta, scale);
    const auto out = rule_forward(x, s0, false);
    return {out[0], out[1]};
}

void check_index(const char* what, const Tensor& t, int64_t B) {
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == B, what,
                      " must have shape (", B, ",), got ",
                      shape_of(t.sizes()));
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong ||
                         t.scalar_type() == at::kInt,
                     what, " must be int64 or int32, got ", t.scalar_type());
}

Tensor gated_delta_step(const Tensor& q, const Tensor& k, const Tensor& v,
                        const Tensor& g, const Tensor& beta,
                        const Tensor& state, const OptTensor& lengths_,
                        const OptTensor& slots_, std::optional<double> scale,
                        bool update) {
    Inputs x(q, k, v, g, beta, scale);
    Tensor lengths = or_undefined(lengths_), slots = or_undefined(slots_);
    no_tangents("gated_delta_step", {&q, &k, &v, &g, &beta, &state});
    TORCH_CHECK(!wants_grad({&q, &k, &v, &g, &beta, &state}),
                "gated_delta_step has no gradient; call it under no_grad, or "
                "gated_delta_rule");
    TORCH_CHECK_VALUE(state.dim() == 4 && state.size(1) == x.in.Hv &&
                          state.size(2) == x.in.Dv &&
                          state.size(3) == x.in.Dk,
                      "state must have shape (pool, ", x.in.Hv, ", ", x.in.Dv,
                      ", ", x.in.Dk, "), got ", shape_of(state.sizes()));
    TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat,
                     "state must be float32, got ", state.scalar_type());
    TORCH_CHECK_VALUE(state.is_contiguous(),
                      "state must be contiguous: it is updated in place");
    if (lengths.defined()) check_index("lengths", lengths, x.in.B);
    if (slots.defined())
        check_index("slots", slots, x.in.B);
    else
        TORCH_CHECK_VALUE(state.size(0) == x.in.B, "a state for each of the ",
                          x.in.B, " rows is needed where slots is None, got ",
                          state.size(0));
    same_gpu({&x.q, &x.k, &x.v, &x.g, &x.beta, &state, &lengths, &slots});
    const c10::DeviceGuard guard(x.q.device());
    x.place();
    const auto ids = [](const Tensor& t) {
        return t.defined() ? t.to(at::kLong).contiguous() : t;
    };
    lengths = ids(lengths);
    slots = ids(slots);
    Tensor o = at::empty(x.o_shape(), x.q.options().requires_grad(false));
    check("rwkv7m_gated_delta_step",
          rwkv7m_gated_delta_step(&x.in, state.size(0), ptr<float>(state),
                                  ptr<int64_t>(slots), ptr<int64_t>(lengths),
                                  update, ptr(o), stream_of(x.q)));
    // (a backward that saved the states as they were has to notice)
    if (update && !state.is_inference())
        state.unsafeGetTensorImpl()->bump_version();
    return o;
}

}  // namespace

void bind_gated_delta(pybind11::module_& m) {
    const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("gated_delta_rule", &gated_delta_rule, free);
    m.def("gated_delta_step", &gated_delta_step, free);
}
