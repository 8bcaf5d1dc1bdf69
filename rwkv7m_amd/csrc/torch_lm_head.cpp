// torch binding of the operators around a language model's head
// (include/rwkv7m_lm_head.h): argument checks, outputs from torch's allocator,
// the current stream, and the autograd nodes.  Host code only; the kernels are
// librwkv7m_wkv.so's.
//
// It is compiled because these calls are short: an autograd node in Python
// and a ctypes call cost a norm's training step at [4096, 768] 125 us of host
// time for 16 us of kernels.

#include "../../include/rwkv7m_lm_head.h"
#include "torch_common.h"

namespace {

// --- layer norm -------------------------------------------------------------

int norm_params(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    const int64_t C = x.size(-1);
    int code = RWKV7M_DTYPE_F32;
    const Tensor* both[2] = {&weight, &bias};
    const char* names[2] = {"weight", "bias"};
    for (int i = 0; i < 2; ++i) {
        if (!both[i]->defined()) continue;
        TORCH_CHECK_VALUE(both[i]->dim() == 1 && both[i]->size(0) == C,
                          names[i], " must have shape (", C, ",), got ",
                          shape_of(both[i]->sizes()));
        code = code_of(names[i], *both[i]);
    }
    TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() ||
                         weight.scalar_type() == bias.scalar_type(),
                     "weight and bias must share one dtype, got ",
                     weight.scalar_type(), " and ", bias.scalar_type());
    return code;
}

// (y, statistics [2, rows] or undefined: mean and rstd)
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight,
                                        const Tensor& bias, double eps,
                                        bool with_stats) {
    const int64_t C = row_width("x", x);
    const int code = code_of("x", x), pcode = norm_params(x, weight, bias);
    same_gpu({&x, &weight, &bias});
    const c10::DeviceGuard guard(x.device());
    const Rows r(x);
    const Tensor w = dense(weight), b = dense(bias);
    Tensor y = at::empty(x.sizes(), x.options().requires_grad(false)), stats;
    if (with_stats) stats = at::empty({2, r.rows()}, f32(x));
    float* mean = ptr<float>(stats);
    check("rwkv7m_layer_norm",
          rwkv7m_layer_norm(code, pcode, r.outer, r.inner, C, r.outer_stride,
                            r.inner_stride, ptr(r.t), ptr(w), ptr(b), eps,
                            ptr(y), mean, mean ? mean + r.rows() : nullptr,
                            stream_of(x)));
    return {y, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const OptTensor& weight, const OptTensor& bias,
                          double eps) {
        const Tensor w = or_undefined(weight), b = or_undefined(bias);
        auto [y, stats] = norm_forward(x, w, b, eps, true);
        ctx->save_for_backward({x, w, b, stats});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        no_tangents("layer_norm", {&dys[0]});
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &bias = saved[2], &stats = saved[3];
        const c10::DeviceGuard guard(x.device());
        const Rows r(x);
        const Tensor w = dense(saved[1]), dy = dys[0].contiguous();
        const int64_t C = x.size(-1), rows = r.rows();
        // (an absent parameter has no edge)
        size_t edge = 1;
        const bool want_w = w.defined() && ctx->needs_input_grad(edge++);
        const bool want_b = bias.defined() && ctx->needs_input_grad(edge);
        Tensor dx, dw, db, ws;
        if (ctx->needs_input_grad(0))
            dx = at::empty(x.sizes(), x.options().requires_grad(false));
        int64_t floats = 0;
        if (want_w) dw = at::empty({C}, w.options().requires_grad(false));
        if (want_b) db = at::empty({C}, bias.options().requires_grad(false));
        if (want_w || want_b) {
            floats = rwkv7m_layer_norm_workspace_floats(rows, C);
            ws = at::empty({floats > 0 ? floats : 1}, f32(x));
        }
        const int pcode = w.defined()      ? code_of("weight", w)
                          : bias.defined() ? code_of("bias", bias)
                                           : RWKV7M_DTYPE_F32;
        const float* mean = ptr<float>(stats);
        check("rwkv7m_layer_norm_backward",
              rwkv7m_layer_norm_backward(
                  code_of("x", x), pcode, r.outer, r.inner, C, r.outer_stride,
                  r.inner_stride, ptr(r.t), ptr(w), mean, mean + rows,
                  ptr(dy), ptr(dx), ptr(dw), ptr(db), ptr<float>(ws), floats,
                  stream_of(x)));
        return once("layer_norm", {dx, dw, db, Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight,
                  const OptTensor& bias, double eps) {
    const Tensor w = or_undefined(weight), b = or_undefined(bias);
    no_tangents("layer_norm", {&x, &w, &b});
    if (!wants_grad({&x, &w, &b}))
        return std::get<0>(norm_forward(x, w, b, eps, false));
    return LayerNorm::apply(x, weight, bias, eps);
}

// --- token log probabilities ------------------------------------------------

void check_shape(const char* what, const Tensor& t, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.sizes() == shape, what, " must have shape ",
                      shape_of(shape), ", got ", shape_of(t.sizes()));
}

void check_ids(const char* what, const Tensor& t, at::IntArrayRef shape) {
    check_shape(what, t, shape);
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong ||
                         t.scalar_type() == at::kInt,
                     what, " must be int64 or int32, got ", t.scalar_type());
}

// What the kernels take: contiguous int64 ids, contiguous fp32 weights.
Tensor ids64(const Tensor& t) { return t.to(at::kLong).contiguous(); }

Tensor weights32(const Tensor& t) {
    return t.defined() ? t.detach().to(at::kFloat).contiguous() : t;
}

// [logprobs, entropy, top_ids, top_logprobs, statistics]; the ids and their
// logprobs undefined with top_k 0, the statistics where not wanted
variable_list score_forward(const Tensor& logits, const Tensor& tokens_,
                            int64_t top_k, double temperature,
                            bool with_stats) {
    const int64_t V = row_width("logits", logits);
    const int code = code_of("logits", logits);
    const auto shape = logits.sizes().slice(0, logits.dim() - 1);
    check_ids("tokens", tokens_, shape);
    same_gpu({&logits, &tokens_});
    const int64_t most = std::min<int64_t>(V, RWKV7M_MAX_TOP_K);
    TORCH_CHECK_VALUE(top_k >= 0 && top_k <= most, "top_k must be within 0 "
                      "and ", most, " (V=", V, "), got ", top_k);
    const c10::DeviceGuard guard(logits.device());
    const Tensor tokens = ids64(tokens_);
    const Rows r(logits);
    const auto opts = f32(logits);
    Tensor lp = at::empty(shape, opts), ent = at::empty(shape, opts), ids, top,
           stats;
    if (top_k) {
        std::vector<int64_t> wide(shape.begin(), shape.end());
        wide.push_back(top_k);
        ids = at::empty(wide, opts.dtype(at::kLong));
        top = at::empty(wide, opts);
    }
    if (with_stats) stats = at::empty({r.rows(), 2}, opts);
    check("rwkv7m_token_logprobs",
          rwkv7m_token_logprobs(
              code, r.outer, r.inner, V, r.outer_stride, r.inner_stride,
              ptr(r.t), ptr<int64_t>(tokens), top_k, temperature,
              ptr<float>(lp), ptr<float>(ent), ptr<int64_t>(ids),
              ptr<float>(top), ptr<float>(stats), stream_of(logits)));
    return {lp, ent, ids, top, stats};
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                                 const Tensor& tokens, int64_t top_k,
                                 double temperature) {
        auto out = score_forward(logits, tokens, top_k, temperature, true);
        ctx->save_for_backward({logits, tokens, out[4], out[1]});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        if (!top_k) return {out[0], out[1]};
        ctx->mark_non_differentiable({out[2], out[3]});
        return {out[0], out[1], out[2], out[3]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        if (!d[0].defined() && !d[1].defined())
            return {Tensor(), Tensor(), Tensor(), Tensor()};
        no_tangents("token_logprobs", {&d[0], &d[1]});
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &stats = saved[2], &ent = saved[3];
        const c10::DeviceGuard guard(logits.device());
        const Tensor tokens = ids64(saved[1]);
        const Tensor dlp = weights32(d[0]), dent = weights32(d[1]);
        const Rows r(logits);
        Tensor dx = at::empty(logits.sizes(),
                              logits.options().requires_grad(false));
        check("rwkv7m_token_logprobs_backward",
              rwkv7m_token_logprobs_backward(
                  code_of("logits", logits), r.outer, r.inner,
                  logits.size(-1), r.outer_stride, r.inner_stride, ptr(r.t),
                  ptr<int64_t>(tokens),
                  ctx->saved_data["temperature"].toDouble(),
                  ptr<float>(stats), ptr<float>(ent), ptr<float>(dlp),
                  ptr<float>(dent), ptr(dx), stream_of(logits)));
        return once("token_logprobs", {dx, Tensor(), Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor, OptTensor, OptTensor> token_logprobs(
    const Tensor& logits, const Tensor& tokens, int64_t top_k,
    double temperature) {
    no_tangents("token_logprobs", {&logits});
    const auto out = wants_grad({&logits})
                         ? TokenLogprobs::apply(logits, tokens, top_k,
                                                temperature)
                         : score_forward(logits, tokens, top_k, temperature,
                                         false);
    if (!top_k) return {out[0], out[1], std::nullopt, std::nullopt};
    return {out[0], out[1], out[2], out[3]};
}

// --- distillation -----------------------------------------------------------

struct Distill {
    int code, tcode;
    int64_t V, K;
    c10::DeviceGuard guard;
    Tensor ids, teacher, weight;
    Rows r;

    static const Tensor& checked(const Tensor& logits, const Tensor& ids,
                                 const Tensor& teacher, const Tensor& weight) {
        row_width("logits", logits);
        code_of("logits", logits);
        const auto shape = logits.sizes().slice(0, logits.dim() - 1);
        TORCH_CHECK_VALUE(
            teacher.dim() == logits.dim() &&
                teacher.sizes().slice(0, teacher.dim() - 1) == shape,
            "teacher_logits must have shape ", shape_of(shape),
            " with K alternatives behind, got ", shape_of(teacher.sizes()));
        TORCH_CHECK_VALUE(teacher.size(-1) <= RWKV7M_MAX_TEACHER_K, "at most ",
                          RWKV7M_MAX_TEACHER_K, " teacher alternatives are "
                          "supported, got ", teacher.size(-1));
        code_of("teacher_logits", teacher);
        check_ids("teacher_ids", ids, teacher.sizes());
        if (weight.defined()) check_shape("weight", weight, shape);
        same_gpu({&logits, &ids, &teacher, &weight});
        return logits;
    }
    Distill(const Tensor& logits, const Tensor& ids_, const Tensor& teacher_,
            const Tensor& weight_)
        : code(code_of("logits", checked(logits, ids_, teacher_, weight_))),
          tcode(code_of("teacher_logits", teacher_)),
          V(logits.size(-1)),
          K(teacher_.size(-1)),
          guard(logits.device()),
          ids(ids64(ids_)),
          teacher(teacher_.contiguous()),
          weight(weights32(weight_)),
          r(logits) {}
};

// [loss, row losses, gradient or undefined]
variable_list distill_forward(const Tensor& logits, const Tensor& ids,
                              const Tensor& teacher, const Tensor& weight,
                              double temperature, bool with_grad) {
    const Distill d(logits, ids, teacher, weight);
    Tensor loss = at::empty({}, f32(logits));
    Tensor rows = at::empty(logits.sizes().slice(0, logits.dim() - 1),
                            f32(logits));
    Tensor dx;
    if (with_grad)
        dx = at::empty(logits.sizes(), logits.options().requires_grad(false));
    check("rwkv7m_distill_loss",
          rwkv7m_distill_loss(d.code, d.tcode, d.r.outer, d.r.inner, d.V,
                              d.r.outer_stride, d.r.inner_stride, d.K,
                              ptr(d.r.t), ptr<int64_t>(d.ids), ptr(d.teacher),
                              ptr<float>(d.weight), temperature,
                              ptr<float>(loss), ptr<float>(rows), ptr(dx),
                              stream_of(logits)));
    return {loss, rows, dx};
}

// The forward writes the gradient too (the logits are read once); the backward
// hands it on where the loss's own cotangent is 1, which the kernel sees on
// the device, and otherwise has it formed anew.
struct DistillLoss : torch::autograd::Function<DistillLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                                 const Tensor& ids, const Tensor& teacher,
                                 const OptTensor& weight, double temperature) {
        const Tensor w = or_undefined(weight);
        auto out = distill_forward(logits, ids, teacher, w, temperature, true);
        ctx->save_for_backward({logits, ids, teacher, w});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["gradient"] = out[2];
        ctx->mark_non_differentiable({out[1]});
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list none(5);
        if (!g[0].defined()) return none;
        no_tangents("distill_loss", {&g[0]});
        const auto saved = ctx->get_saved_variables();
        const Tensor& logits = saved[0];
        const Distill d(logits, saved[1], saved[2], saved[3]);
        const Tensor scale = weights32(g[0]);
        // a second backward over a retained graph gets a buffer of its own
        Tensor dx;
        const auto kept = ctx->saved_data.find("gradient");
        const bool held = kept != ctx->saved_data.end();
        if (held) {
            dx = kept->second.toTensor();
            ctx->saved_data.erase(kept);
        } else {
            dx = at::empty(logits.sizes(),
                           logits.options().requires_grad(false));
        }
        check("rwkv7m_distill_loss_backward",
              rwkv7m_distill_loss_backward(
                  d.code, d.tcode, d.r.outer, d.r.inner, d.V,
                  d.r.outer_stride, d.r.inner_stride, d.K, ptr(d.r.t),
                  ptr<int64_t>(d.ids), ptr(d.teacher), ptr<float>(d.weight),
                  ctx->saved_data["temperature"].toDouble(),
                  ptr<float>(scale), held, ptr(dx), stream_of(logits)));
        none[0] = dx;
        return once("distill_loss", std::move(none));
    }
};

std::tuple<Tensor, Tensor> distill_loss(const Tensor& logits,
                                        const Tensor& ids,
                                        const Tensor& teacher,
                                        const OptTensor& weight,
                                        double temperature) {
    const Tensor w = or_undefined(weight);
    no_tangents("distill_loss", {&logits, &teacher, &w});
    const auto out =
        wants_grad({&logits})
            ? DistillLoss::apply(logits, ids, teacher, weight, temperature)
            : distill_forward(logits, ids, teacher, w, temperature, false);
    return {out[0], out[1]};
}

// --- verification of drafted tokens -----------------------------------------

// Random numbers as the kernels take them, of the given shape.
Tensor uniforms(const char* what, const OptTensor& t, at::IntArrayRef shape,
                const Tensor& like) {
    TORCH_CHECK_VALUE(t && t->defined(), what,
                      " are needed where temperature is not 0");
    check_shape(what, *t, shape);
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, what,
                     " must be float32, got ", t->scalar_type());
    same_gpu({&like, &*t});
    return t->detach().contiguous();
}

std::tuple<Tensor, Tensor, Tensor> verify_drafts(
    const Tensor& logits, const Tensor& tokens_, const OptTensor& draft_,
    const OptTensor& accept_, const OptTensor& sample_,
    const OptTensor& lengths_, double temperature) {
    const int code = code_of("logits", logits);
    TORCH_CHECK_VALUE(logits.dim() == 3 && logits.size(1) >= 1 &&
                          logits.size(2) >= 1,
                      "logits must have shape (B, K + 1, V), got ",
                      shape_of(logits.sizes()));
    const int64_t B = logits.size(0), K = logits.size(1) - 1,
                  V = logits.size(2);
    TORCH_CHECK_VALUE(K <= RWKV7M_MAX_DRAFTS, "at most ", RWKV7M_MAX_DRAFTS,
                      " drafts are supported, got ", K);
    check_ids("draft_tokens", tokens_, {B, K});
    Tensor draft = or_undefined(draft_), lengths = or_undefined(lengths_);
    if (draft.defined()) {
        check_shape("draft_logits", draft, {B, K, V});
        TORCH_CHECK_TYPE(draft.scalar_type() == logits.scalar_type(),
                         "logits and draft_logits must share one dtype, got ",
                         logits.scalar_type(), " and ", draft.scalar_type());
    }
    if (lengths.defined()) check_ids("draft_lengths", lengths, {B});
    const Tensor given[2] = {or_undefined(accept_), or_undefined(sample_)};
    no_tangents("verify_drafts", {&logits, &draft, &given[0], &given[1]});
    TORCH_CHECK(!wants_grad({&logits, &draft, &given[0], &given[1]}),
                "verify_drafts has no gradient; call it under no_grad, or on "
                "detached logits");
    same_gpu({&logits, &tokens_, &draft, &lengths});
    const bool greedy = temperature == 0.0;
    Tensor accept, sample;
    if (!greedy) {
        accept = uniforms("accept_uniforms", accept_, {B, K}, logits);
        sample = uniforms("sample_uniforms", sample_, {B}, logits);
    }
    const c10::DeviceGuard guard(logits.device());
    const Tensor tokens = ids64(tokens_);
    if (lengths.defined()) lengths = ids64(lengths);
    const auto opts = f32(logits);
    Tensor out = at::empty({B, K + 1}, opts.dtype(at::kLong));
    Tensor accepted = at::empty({B}, opts.dtype(at::kLong));
    Tensor chances = at::empty({B, K}, opts);
    // rows of two axes: batch and position
    const auto rows = [](const Tensor& t, int64_t stride[2]) -> Tensor {
        const bool fits = t.size(2) == 1 || t.stride(2) == 1;
        const Tensor dense_ = fits ? t : t.contiguous();
        for (int i = 0; i < 2; ++i)
            stride[i] = t.size(i) > 1 ? dense_.stride(i) : 0;
        return dense_;
    };
    int64_t ts[2] = {0, 0}, ds[2] = {0, 0};
    const Tensor target = rows(logits, ts);
    if (draft.defined() && K > 0) draft = rows(draft, ds);
    const int64_t bytes = rwkv7m_verify_drafts_workspace_bytes(B, K, V);
    const Tensor ws =
        at::empty({bytes > 0 ? bytes : 1}, opts.dtype(at::kByte));
    check("rwkv7m_verify_drafts",
          rwkv7m_verify_drafts(
              code, B, K, V, ts[0], ts[1], ptr(target), ds[0], ds[1],
              K > 0 ? ptr(draft) : nullptr, ptr<int64_t>(tokens),
              ptr<float>(accept), ptr<float>(sample), ptr<int64_t>(lengths),
              temperature, ptr<int64_t>(out), ptr<int64_t>(accepted),
              ptr<float>(chances), ptr(ws), bytes, stream_of(logits)));
    return {out, accepted, chances};
}

}  // namespace

void bind_gated_delta(pybind11::module_& m);  // torch_gated_delta.cpp

PYBIND11_MODULE(_lm_head_torch, m) {
    const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("layer_norm", &layer_norm, free);
    m.def("token_logprobs", &token_logprobs, free);
    m.def("distill_loss", &distill_loss, free);
    m.def("verify_drafts", &verify_drafts, free);
    bind_gated_delta(m);
}
