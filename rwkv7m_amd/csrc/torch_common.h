// What the torch bindings share (torch_lm_head.cpp, torch_gated_delta.cpp):
// checks of arguments, the current stream, and gradients of first order.  Host
// code only.
#pragma once

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/rwkv7m_wkv.h"

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

}  // namespace
