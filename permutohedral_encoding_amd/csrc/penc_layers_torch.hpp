// What the layers' sources of the extension _penc_torch share: checks of tensors, rows of adjacent channels, and the node of autograd that theirs derive from.
#pragma once

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <memory>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "../../include/penc.h"
#include "penc_torch.hpp"

namespace penc_torch {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline int type_of(at::ScalarType t, const char* name) {
    switch (t) {
        case at::kFloat: return PENC_FP32;
        case at::kHalf: return PENC_FP16;
        case at::kBFloat16: return PENC_BF16;
        default: PENC_REQUIRE(false, name, " should be of type float32, float16 or bfloat16, however it is ", t);
    }
    return -1;
}
inline at::ScalarType scalar_type_of(long code) {
    PENC_REQUIRE(code == PENC_FP32 || code == PENC_FP16 || code == PENC_BF16, "no such type");
    return code == PENC_FP32 ? at::kFloat : code == PENC_FP16 ? at::kHalf : at::kBFloat16;
}

// The kernels write and read through pointers: what has to see tensor operations instead is refused.
inline void require_plain(std::initializer_list<const Tensor*> tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
                                    !torch::jit::tracer::isTracing(),
                                "the layers have no rule for functorch transforms and traces");
    const Tensor* first = nullptr;
    for (const Tensor* t : tensors) {
        if (!t->defined()) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), "forward-mode differentiation of the layers is not implemented");
        PENC_REQUIRE(t->is_cuda(), "the layers' tensors should be in GPU memory. Please call .cuda() on the tensor");
        PENC_REQUIRE(t->layout() == at::kStrided && !t->is_neg() && !t->_is_zerotensor(), "the layers take dense tensors that are in memory as they are");
        if (first == nullptr) first = t;
        PENC_REQUIRE(t->device() == first->device(), "the layers' tensors must be on the same device");
    }
}

// A tensor (..., C) as rows of adjacent channels, `stride` values apart: itself where it can be read so, else a copy.
struct Rows {
    Tensor values;
    int64_t n = 0, channels = 0, stride = 0;
    const void* data() const { return values.const_data_ptr(); }
};

// Whether the leading dimensions are one dimension of rows, and how far apart those are.
inline bool rows_in_place(const Tensor& t, int64_t& stride) {
    const int64_t d = t.dim(), channels = t.size(d - 1);
    if (t.stride(d - 1) != 1 && channels != 1) return false;
    stride = channels;
    int64_t next = -1;
    for (int64_t i = d - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (next < 0) stride = t.stride(i);
        else if (t.stride(i) != next) return false;
        next = t.stride(i) * t.size(i);
    }
    return true;
}

inline Rows rows_of(const Tensor& t, const char* name) {
    PENC_REQUIRE(t.dim() >= 1, name, " should have channels, however it has no dimension");
    Rows r;
    r.channels = t.size(-1);
    PENC_REQUIRE(r.channels >= 1, name, " should have at least one channel, however it has sizes ", t.sizes());
    r.n = t.numel() / r.channels;
    r.values = t;
    if (r.n == 0) {
        r.stride = r.channels;
    } else if (!rows_in_place(t, r.stride) || r.stride >= (int64_t{1} << 31)) {
        r.values = t.contiguous();
        r.stride = r.channels;
    }
    return r;
}

inline Tensor empty_rows(const Tensor& like, int64_t channels) {
    std::vector<int64_t> sizes = like.sizes().vec();
    sizes.back() = channels;
    return at::empty(sizes, like.options());
}

inline bool any_requires_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// What the nodes share: tensors saved for the backward, and the refusal to differentiate it.
struct LayerNode : public Node {
    std::vector<SavedVariable> saved;

    void save(std::initializer_list<const Tensor*> tensors) {
        saved.reserve(tensors.size());
        for (const Tensor* t : tensors) saved.emplace_back(t->defined() ? SavedVariable(*t, false) : SavedVariable());
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        for (SavedVariable& s : saved) s.reset_data();
    }
    std::vector<Tensor> unpacked() {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        std::vector<Tensor> t;
        t.reserve(saved.size());
        for (SavedVariable& s : saved) t.push_back(s.unpack(shared_from_this()));
        return t;
    }
    variable_list apply(variable_list&& grads) override {
        bool any = false;
        for (Tensor& g : grads) {
            if (!g.defined()) continue;
            any = true;
            if (g.is_neg()) {  // (the imaginary part of a conjugated gradient, for instance: negated when it is read)
                at::NoGradGuard no_grad;
                g = g.resolve_neg();
            }
            require_plain({&g});
        }
        if (!any) return variable_list(num_outputs());
        const bool differentiable = at::GradMode::is_enabled();
        variable_list out;
        {
            at::NoGradGuard no_grad;
            out = gradients(grads);
        }
        if (differentiable) {
            // (with create_graph: whoever differentiates these is told, and does not get a zero)
            for (Tensor& t : out)
                if (t.defined()) t.set_requires_grad(true);
            auto refusal = std::make_shared<torch::autograd::DelayedError>(
                std::string("the gradients of the layers cannot be differentiated again: ") + why_once(), static_cast<int64_t>(out.size()));
            out = (*refusal)(std::move(out));
        }
        return out;
    }
    virtual variable_list gradients(const variable_list& grads) = 0;
    virtual const char* why_once() const { return "what they keep in 8 bits has no second derivative"; }

private:
    bool released = false;
};

template <class N>
std::shared_ptr<N> make_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

inline void require_saved(const Tensor& t, c10::IntArrayRef sizes, at::ScalarType type) {
    TORCH_CHECK(t.defined() && t.is_cuda() && t.sizes() == sizes && t.scalar_type() == type, "a tensor saved for the backward has come back in another form");
}

// The gradient of a result as rows of the result's type (autograd has brought it to the result's sizes).
inline Rows grad_rows(const Tensor& g, at::ScalarType type) { return rows_of(g.scalar_type() == type ? g.detach() : g.detach().to(type), "the gradient"); }

// ---- Python

inline Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }

template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name, const char* doc) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFunction)), METH_FASTCALL, doc};
}

}  // namespace penc_torch
