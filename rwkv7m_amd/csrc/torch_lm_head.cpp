// torch binding of the operators around a language model's head
// (include/rwkv7m_lm_head.h): argument checks, outputs from torch's allocator,
// the current stream, and the autograd nodes.  Host code only; the kernels are
// librwkv7m_wkv.so's.
//
// It is compiled because these calls are short: an autograd node in Python
// and a ctypes call cost a norm's training step at [4096, 768] 125 us of host
// time for 16 us of kernels.

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/rwkv7m_lm_head.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

std::string shape_of(at::IntArrayRef s) {
    std::string out = "(";
    for (size_t i = 0; i < s.size(); ++i)
        out += (i ? ", " : "") + std::to_string(s[i]);
    return out + (s.size() == 1 ? ",)" : ")");
}

int code_of(const char* what, const Tensor& t) {
    const auto type = t.scalar_type();
    TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16, what,
                     " must be bfloat16 or float32, got ", type);
    return type == at::kFloat ? RWKV7M_DTYPE_F32 : RWKV7M_DTYPE_BF16;
}

int64_t row_width(const char* what, const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, what,
                      " must have at least one element along its last axis, "
                      "got shape ",
                      shape_of(t.sizes()));
    return t.size(-1);
}

// Every defined tensor is on the first one's GPU.
void same_gpu(std::initializer_list<const Tensor*> tensors) {
    const Tensor* first = nullptr;
    for (const Tensor* t : tensors) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->is_cuda(), "the HIP kernels need GPU tensors; got a "
                    "tensor on ", t->device(), " (there is no CPU fallback)");
        if (!first) first = t;
        TORCH_CHECK(t->device() == first->device(),
                    "all tensors must be on one device, got ",
                    first->device(), " and ", t->device());
    }
}

void check(const char* fn, int rc) {
    TORCH_CHECK(rc == RWKV7M_OK, fn, " failed (status ", rc, "): ",
                rwkv7m_last_error());
}

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// The rows along the last axis: `t` where it lies, if its leading axes are
// one or two strided ones once adjoining axes are merged, else a copy.
struct Rows {
    Tensor t;
    int64_t outer = 1, inner, outer_stride = 0, inner_stride;

    explicit Rows(const Tensor& from) : t(from) {
        const int64_t n = t.size(-1);
        inner = t.numel() / n;
        inner_stride = n;
        if (t.is_contiguous()) return;
        int64_t size[2] = {1, 1}, stride[2] = {0, 0};
        int axes = 0;
        bool fits = n == 1 || t.stride(-1) == 1;
        for (int64_t a = t.dim() - 2; a >= 0 && fits; --a) {
            if (t.size(a) == 1) continue;
            if (axes && t.stride(a) == size[axes - 1] * stride[axes - 1]) {
                size[axes - 1] *= t.size(a);
            } else if (axes < 2) {
                size[axes] = t.size(a);
                stride[axes++] = t.stride(a);
            } else {
                fits = false;
            }
        }
        if (!fits) {
            t = t.contiguous();
            return;
        }
        inner = size[0];
        inner_stride = stride[0];
        outer = size[1];
        outer_stride = stride[1];
    }
    int64_t rows() const { return outer * inner; }
};

Tensor or_undefined(const OptTensor& t) { return t ? *t : Tensor(); }

Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// A tangent of forward-mode differentiation, which needs no gradient to be
// enabled, is refused and not dropped.
void no_tangents(const char* fn, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK_TYPE(!t->defined() || !t->_fw_grad(0).defined(), fn,
                         " supports reverse-mode differentiation only; "
                         "forward-mode autodiff (jvp) is not implemented");
}

at::TensorOptions f32(const Tensor& like) {
    return like.options().dtype(at::kFloat).requires_grad(false);
}

// Gradients are first order: where a graph of the backward is asked for, they
// join it with an error for whoever differentiates them.
variable_list once(const char* fn, variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list defined;
    for (auto& g : grads)
        if (g.defined()) defined.push_back(g.detach().requires_grad_());
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(fn) + " is once_differentiable: its gradient has none",
        int64_t(defined.size()));
    variable_list out = (*error)(std::move(defined));
    size_t at = 0;
    for (auto& g : grads)
        if (g.defined()) g = out[at++];
    return grads;
}

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

}  // namespace

PYBIND11_MODULE(_lm_head_torch, m) {
    const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("layer_norm", &layer_norm, free);
    m.def("token_logprobs", &token_logprobs, free);
    m.def("distill_loss", &distill_loss, free);
}
