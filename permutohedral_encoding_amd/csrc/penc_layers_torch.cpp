// The path from the functions of layers.py to the kernels and back through autograd, in native code, as penc_torch.cpp has it for the
// encoding: one call into this extension, and autograd nodes that never enter the interpreter.
//
// What a node keeps of its inputs in 8 bits it saves as autograd saves tensors (freed with the graph, seen by saved-tensor hooks);
// parameters are saved themselves, with the version checks that go with it.  Gradients are those of the operators at the values kept, and cannot be
// differentiated again.
#include <ATen/SavedTensorHooks.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <dlfcn.h>
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

namespace {

using namespace penc_torch;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Api {
#define PENC_FN(name) decltype(&penc_##name) name = nullptr
    PENC_FN(status_string);
    PENC_FN(kept_pitch);
    PENC_FN(kept_blocks);
    PENC_FN(keep);
    PENC_FN(restore);
    PENC_FN(activation);
    PENC_FN(activation_backward);
    PENC_FN(weight_grad_workspace_bytes);
    PENC_FN(weight_grad);
    PENC_FN(residual_norm);
    PENC_FN(residual_norm_workspace_bytes);
    PENC_FN(residual_norm_backward);
#undef PENC_FN
} api;

void check(int status, const char* what) {
    if (status != PENC_OK) TORCH_CHECK(false, what, ": ", api.status_string(status), " (status ", status, ")");
}

int type_of(at::ScalarType t, const char* name) {
    switch (t) {
        case at::kFloat: return PENC_FP32;
        case at::kHalf: return PENC_FP16;
        case at::kBFloat16: return PENC_BF16;
        default: PENC_REQUIRE(false, name, " should be of type float32, float16 or bfloat16, however it is ", t);
    }
    return -1;
}
at::ScalarType scalar_type_of(long code) {
    PENC_REQUIRE(code == PENC_FP32 || code == PENC_FP16 || code == PENC_BF16, "no such type");
    return code == PENC_FP32 ? at::kFloat : code == PENC_FP16 ? at::kHalf : at::kBFloat16;
}

// The kernels write and read through pointers: what has to see tensor operations instead is refused.
void require_plain(std::initializer_list<const Tensor*> tensors) {
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
bool rows_in_place(const Tensor& t, int64_t& stride) {
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

Rows rows_of(const Tensor& t, const char* name) {
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

Tensor empty_rows(const Tensor& like, int64_t channels) {
    std::vector<int64_t> sizes = like.sizes().vec();
    sizes.back() = channels;
    return at::empty(sizes, like.options());
}

// ------------------------------------------------------------------------------------------
// checkpoints

// `count` checkpoints of rows in one piece of memory: the values of each, one behind the other, then the exponents of each.
struct Checkpoint {
    Tensor bytes;  // int8; undefined: none
    int64_t rows = 0, channels = 0, count = 1;

    int8_t* q(int64_t k = 0) const { return bytes.defined() ? static_cast<int8_t*>(bytes.data_ptr()) + k * rows * api.kept_pitch(channels) : nullptr; }
    uint8_t* e(int64_t k = 0) const {
        return bytes.defined() ? reinterpret_cast<uint8_t*>(q(count)) + k * rows * api.kept_blocks(channels) : nullptr;
    }
    static int64_t size(int64_t rows, int64_t channels, int64_t count) { return count * rows * (api.kept_pitch(channels) + api.kept_blocks(channels)); }
};

Checkpoint room_for(const Tensor& like, int64_t rows, int64_t channels, int64_t count = 1) {
    return {at::empty({Checkpoint::size(rows, channels, count)}, like.options().dtype(at::kChar)), rows, channels, count};
}

Checkpoint keep(const Tensor& x, const char* name) {
    const int type = type_of(x.scalar_type(), name);
    PENC_REQUIRE(x.dim() >= 1 && x.size(-1) >= 1, name, " should have at least one channel, however it has sizes ", x.sizes());
    PENC_REQUIRE(x.size(-1) <= PENC_MAX_CHANNELS, name, " has more than ", PENC_MAX_CHANNELS, " channels");
    // the encoding's own result: channels of consecutive rows side by side
    const bool by_channels = x.dim() == 2 && x.size(0) > 1 && x.size(1) > 1 && x.size(1) <= (1 << 22) && x.stride(0) == 1 && x.stride(1) >= x.size(0);
    const Rows r = by_channels ? Rows{x, x.size(0), x.size(1), 1} : rows_of(x, name);
    Checkpoint kept = room_for(x, r.n, r.channels);
    check(api.keep(type, r.n, r.channels, r.data(), r.stride, by_channels ? x.stride(1) : 1, kept.q(), kept.e(), current_stream(x.device())), "checkpoint");
    return kept;
}

std::pair<Tensor, Tensor> weight_grad(const Checkpoint& kept, int64_t channels, const Tensor& grad, at::ScalarType result, bool bias) {
    const int type = type_of(grad.scalar_type(), "grad");
    const Rows g = rows_of(grad, "grad");
    PENC_REQUIRE(g.n == kept.rows, "grad should have a row for each of the ", kept.rows, " rows kept, however it has sizes ", grad.sizes());
    const auto options = grad.options().dtype(result);
    Tensor weight = at::empty({g.channels, channels}, options), b;
    if (bias) b = at::empty({g.channels}, options);
    const size_t n = api.weight_grad_workspace_bytes(g.n, channels, g.channels);
    const Tensor ws = at::empty({static_cast<int64_t>(n)}, grad.options().dtype(at::kByte));
    check(api.weight_grad(type, type_of(result, "weight"), g.n, channels, g.channels, kept.q(), kept.e(), g.data(), g.stride, weight.data_ptr(),
                          bias ? b.data_ptr() : nullptr, ws.data_ptr(), n, current_stream(grad.device())),
          "weight_grad");
    return {weight, b};
}

// ------------------------------------------------------------------------------------------
// autograd

bool any_requires_grad(std::initializer_list<const Tensor*> tensors) {
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
                "the gradients of the layers cannot be differentiated again: what they keep in 8 bits has no second derivative", static_cast<int64_t>(out.size()));
            out = (*refusal)(std::move(out));
        }
        return out;
    }
    virtual variable_list gradients(const variable_list& grads) = 0;

private:
    bool released = false;
};

template <class N>
std::shared_ptr<N> make_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// What hooks on saved tensors may have brought back in another form.
Checkpoint saved_checkpoint(const Tensor& bytes, int64_t rows, int64_t channels, int64_t count) {
    TORCH_CHECK(bytes.defined() && bytes.is_cuda() && bytes.scalar_type() == at::kChar && bytes.is_contiguous() &&
                    bytes.numel() == Checkpoint::size(rows, channels, count),
                "a checkpoint saved for the backward has come back in another form");
    return {bytes, rows, channels, count};
}
void require_saved(const Tensor& t, c10::IntArrayRef sizes, at::ScalarType type) {
    TORCH_CHECK(t.defined() && t.is_cuda() && t.sizes() == sizes && t.scalar_type() == type, "a tensor saved for the backward has come back in another form");
}

// The gradient of a result as rows of the result's type (autograd has brought it to the result's sizes).
Rows grad_rows(const Tensor& g, at::ScalarType type) { return rows_of(g.scalar_type() == type ? g.detach() : g.detach().to(type), "the gradient"); }

// ---- linear

struct LinearNode : public LayerNode {
    int64_t channels = 0;
    std::vector<int64_t> x_sizes;
    at::ScalarType type;
    bool has_bias = false;

    std::string name() const override { return "LayersLinearBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();  // the weight, where x wants a gradient, and the checkpoint of x
        const Tensor g = (grads[0].scalar_type() == type ? grads[0] : grads[0].to(type)).reshape({-1, grads[0].size(-1)});
        const c10::DeviceGuard device(g.device());
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        variable_list out(3);
        if (task_should_compute_output(0)) out[0] = at::mm(g, t[0]).view(x_sizes);
        const bool want_bias = has_bias && task_should_compute_output(2);
        if (t[1].defined() && (task_should_compute_output(1) || want_bias))
            std::tie(out[1], out[2]) = weight_grad(saved_checkpoint(t[1], g.size(0), channels, 1), channels, g, type, want_bias);
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    require_plain({&x, &weight, &bias});
    type_of(x.scalar_type(), "x");
    PENC_REQUIRE(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1) && weight.size(0) >= 1 && weight.size(1) >= 1,
                 "linear should have rows of ", weight.dim() == 2 ? weight.size(1) : -1, " channels, however x has sizes ", x.sizes());
    PENC_REQUIRE(weight.scalar_type() == x.scalar_type() && (!bias.defined() || bias.scalar_type() == x.scalar_type()),
                 "x, weight and bias of linear should be of one type");
    PENC_REQUIRE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0)), "linear should have a bias for each of its outputs");
    const c10::DeviceGuard device(x.device());
    const bool differentiable = any_requires_grad({&x, &weight, &bias});
    Tensor y;
    Checkpoint kept;
    {
        at::NoGradGuard no_grad;
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        // (as rows: of leading dimensions that are not one, at::linear makes a batched product whose right operand is a transposed view, and in 16 bits those
        // have faulted the GPU)
        const Tensor rows = x.dim() == 2 ? x.detach() : x.detach().reshape({-1, x.size(-1)});
        y = at::linear(rows, weight, bias);
        if (x.dim() != 2) {
            std::vector<int64_t> sizes = x.sizes().vec();
            sizes.back() = weight.size(0);
            y = at::_unsafe_view(y, sizes);  // (a result of its own, and no view of one made without gradients)
        }
        // (for the bias alone too: its sum comes with the weight's)
        if (differentiable && (weight.requires_grad() || (bias.defined() && bias.requires_grad()))) kept = keep(rows, "x");
    }
    if (!differentiable) return y;
    auto node = make_node<LinearNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->channels = x.size(-1);
    node->x_sizes = x.sizes().vec();
    node->type = x.scalar_type();
    node->has_bias = bias.defined();
    // (the weight for the gradient of x alone: where x wants none, it may be changed before the backward, as with torch's own layer)
    const Tensor none;
    node->save({x.requires_grad() ? &weight : &none, &kept.bytes});
    torch::autograd::set_history(y, node);
    return y;
}

// ---- activation

struct ActivationNode : public LayerNode {
    int kind = 0, type = 0, gated = 0;
    bool keep_8bit = true;
    int64_t rows = 0, channels = 0;
    std::vector<int64_t> sizes;  // of x

    std::string name() const override { return "LayersActivationBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();  // x, or its checkpoint
        const c10::DeviceGuard device(grads[0].device());
        variable_list out(1);
        out[0] = at::empty(sizes, grads[0].options().dtype(scalar_type_of(type)));
        if (rows == 0) return out;
        const Rows g = grad_rows(grads[0], scalar_type_of(type));
        Rows x;
        Checkpoint kept;
        if (keep_8bit) {
            kept = saved_checkpoint(t[1], rows, channels, gated ? 2 : 1);
        } else {
            require_saved(t[0], sizes, scalar_type_of(type));
            x = rows_of(t[0], "x");
        }
        check(api.activation_backward(type, kind, gated, rows, channels, keep_8bit ? nullptr : x.data(), x.stride, kept.q(), kept.e(), g.data(),
                                      g.stride, out[0].data_ptr(), current_stream(out[0].device())),
              "activation");
        return out;
    }
};

Tensor activation(const Tensor& x, int kind, bool gated, bool keep_8bit) {
    require_plain({&x});
    const int type = type_of(x.scalar_type(), "x");
    const c10::DeviceGuard device(x.device());
    const bool differentiable = any_requires_grad({&x});
    Tensor y;
    Checkpoint kept;
    int64_t rows, channels;
    {
        at::NoGradGuard no_grad;
        const Rows r = rows_of(x.detach(), "x");
        PENC_REQUIRE(!gated || r.channels % 2 == 0, "a gated activation should have two halves of channels, however x has sizes ", x.sizes());
        rows = r.n;
        channels = gated ? r.channels / 2 : r.channels;
        PENC_REQUIRE(channels <= PENC_MAX_CHANNELS, "x has more than ", PENC_MAX_CHANNELS, " channels");
        y = empty_rows(x, channels);
        if (differentiable && keep_8bit) kept = room_for(x, rows, channels, gated ? 2 : 1);
        check(api.activation(type, kind, gated, rows, channels, r.data(), r.stride, y.data_ptr(), kept.q(), kept.e(), current_stream(x.device())),
              "activation");
    }
    if (!differentiable) return y;
    auto node = make_node<ActivationNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->kind = kind, node->type = type, node->gated = gated, node->keep_8bit = keep_8bit;
    node->rows = rows, node->channels = channels;
    node->sizes = x.sizes().vec();
    const Tensor none;
    node->save({keep_8bit ? &none : &x, &kept.bytes});
    torch::autograd::set_history(y, node);
    return y;
}

// ---- residual_norm

// How many consecutive rows share a gate, 0 for one gate for all.
int64_t rows_per_gate(const Tensor& x, const Tensor& gate, int64_t rows, int64_t channels) {
    const auto refuse = [&] {
        PENC_REQUIRE(false, "gate should have sizes (C,), those of x with trailing ones before the channels, or (groups, C) for x of (rows, C), however x has sizes ",
                     x.sizes(), " and gate ", gate.sizes());
    };
    if (gate.dim() < 1 || gate.size(-1) != channels) refuse();
    if (gate.numel() == channels && gate.dim() <= x.dim()) return 0;
    if (gate.dim() != x.dim()) refuse();
    int64_t groups = 1;
    if (x.dim() == 2) {
        groups = gate.size(0);
    } else {
        bool inside = false;  // behind the dimensions that have gates of their own
        for (int64_t i = 0; i + 1 < x.dim(); ++i) {
            if (!inside && gate.size(i) == x.size(i)) {
                groups *= x.size(i);
            } else {
                inside = true;
                if (gate.size(i) != 1) refuse();
            }
        }
    }
    if (groups == 0 ? rows != 0 : rows % groups != 0) refuse();
    return rows == 0 ? 0 : rows / groups;
}

struct NormOptions {
    double scale, eps;
    int kind;
    bool post_norm, pre_norm, keep_8bit;
};

// A norm's arguments without the rows; the parameters' memory has to outlive the call.
penc_norm norm_of(const NormOptions& o, int type, int64_t rows, int64_t channels, int64_t per_gate, const Tensor& gate, const Tensor (&params)[4]) {
    penc_norm n{};
    n.type = n.param_type = n.gate_type = type;
    if (gate.defined()) n.gate_type = type_of(gate.scalar_type(), "gate");
    for (const Tensor& p : params)
        if (p.defined()) n.param_type = type_of(p.scalar_type(), "weight");
    n.kind = o.kind;
    n.post_norm = o.post_norm, n.pre_norm = o.pre_norm;
    n.residual_scale = static_cast<float>(o.scale), n.eps = static_cast<float>(o.eps);
    n.rows = rows, n.channels = channels, n.rows_per_gate = per_gate;
    const auto at = [](const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; };
    n.gate = at(gate);
    n.post_weight = at(params[0]), n.post_bias = at(params[1]), n.pre_weight = at(params[2]), n.pre_bias = at(params[3]);
    return n;
}

struct NormNode : public LayerNode {
    NormOptions options;
    int type = 0;
    int64_t rows = 0, channels = 0, per_gate = 0;
    bool has_branch = false, has_y = false;
    std::vector<int64_t> sizes, param_sizes[5];  // of x; of the gate, weights and biases
    at::ScalarType param_types[5] = {};

    std::string name() const override { return "LayersResidualNormBackward"; }
    variable_list gradients(const variable_list& grads) override {
        // x and branch, or (undefined) the checkpoints of both, gate, post weight and bias, pre weight and bias
        const std::vector<Tensor> t = unpacked();
        const auto scalar = scalar_type_of(type);
        for (int i = 0; i < 5; ++i) {
            TORCH_CHECK(t[3 + i].defined() == (param_sizes[i].size() != 0), "a parameter saved for the backward has not come back");
            if (t[3 + i].defined()) require_saved(t[3 + i], param_sizes[i], param_types[i]);
        }
        const Tensor gate = t[3].defined() ? t[3].contiguous() : Tensor();
        Tensor params[4];
        for (int i = 0; i < 4; ++i)
            if (t[4 + i].defined()) params[i] = t[4 + i].contiguous();
        const Tensor& any = grads[0].defined() ? grads[0] : grads[1];
        const c10::DeviceGuard device(any.device());
        variable_list out(7);
        const auto options_of_rows = any.options().dtype(scalar);
        if (task_should_compute_output(0)) out[0] = at::empty(sizes, options_of_rows);
        if (has_branch && task_should_compute_output(1)) out[1] = at::empty(sizes, options_of_rows);
        for (int i = 0; i < 5; ++i)
            if (t[3 + i].defined() && task_should_compute_output(2 + i)) out[2 + i] = at::empty(t[3 + i].sizes(), t[3 + i].options());
        if (rows == 0) {
            for (Tensor& o : out)
                if (o.defined()) o.zero_();
            return out;
        }
        penc_norm n = norm_of(options, type, rows, channels, per_gate, gate, params);
        n.has_branch = has_branch;
        Rows x, branch, gy, gn;
        if (options.keep_8bit) {
            const Checkpoint kept = saved_checkpoint(t[2], rows, channels, has_branch ? 2 : 1);
            n.x_values = kept.q(), n.x_exponents = kept.e();
            if (has_branch) n.branch_values = kept.q(1), n.branch_exponents = kept.e(1);
        } else {
            require_saved(t[0], sizes, scalar);
            if (has_branch) require_saved(t[1], sizes, scalar);
            x = rows_of(t[0], "x");
            n.x = x.data(), n.x_stride = x.stride;
            if (has_branch) {
                branch = rows_of(t[1], "branch");
                n.branch = branch.data(), n.branch_stride = branch.stride;
            }
        }
        penc_norm_grads g{};
        if (has_y && grads[0].defined()) {
            gy = grad_rows(grads[0], scalar);
            g.y = gy.data(), g.y_stride = gy.stride;
        }
        const Tensor& grad_n = has_y ? grads.back() : grads[0];
        if (options.pre_norm && grad_n.defined()) {
            gn = grad_rows(grad_n, scalar);
            g.n = gn.data(), g.n_stride = gn.stride;
        }
        void** const to[7] = {&g.x, &g.branch, &g.gate, &g.post_weight, &g.post_bias, &g.pre_weight, &g.pre_bias};
        for (int i = 0; i < 7; ++i) *to[i] = out[i].defined() ? out[i].data_ptr() : nullptr;
        const size_t bytes = api.residual_norm_workspace_bytes(rows, channels, per_gate);
        const Tensor ws = at::empty({static_cast<int64_t>(bytes)}, any.options().dtype(at::kByte));
        check(api.residual_norm_backward(&n, &g, ws.data_ptr(), bytes, current_stream(any.device())), "residual_norm");
        return out;
    }
};

// -> y and n; y is undefined without a branch, n without the norm before the next block
std::pair<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& branch, const Tensor& gate, const Tensor (&params)[4], const NormOptions& o) {
    require_plain({&x, &branch, &gate, &params[0], &params[1], &params[2], &params[3]});
    const int type = type_of(x.scalar_type(), "x");
    const bool has_branch = branch.defined();
    const c10::DeviceGuard device(x.device());
    const bool differentiable = any_requires_grad({&x, &branch, &gate, &params[0], &params[1], &params[2], &params[3]});
    Tensor y, n;
    Checkpoint kept;
    int64_t rows, channels, per_gate = 0;
    {
        at::NoGradGuard no_grad;
        const Rows r = rows_of(x.detach(), "x");
        rows = r.n, channels = r.channels;
        PENC_REQUIRE(channels <= PENC_MAX_NORM_CHANNELS, "a row that is normed should have at most ", PENC_MAX_NORM_CHANNELS, " channels, however x has sizes ", x.sizes());
        Rows b;
        if (has_branch) {
            PENC_REQUIRE(branch.sizes() == x.sizes() && branch.scalar_type() == x.scalar_type(),
                         "branch should have the sizes and type of x, however they are ", branch.sizes(), " ", branch.scalar_type(), " and ", x.sizes(), " ",
                         x.scalar_type());
            b = rows_of(branch.detach(), "branch");
        }
        PENC_REQUIRE(has_branch || !gate.defined(), "a gate is for a branch");
        const auto own_or_float = [&](const Tensor& t, const char* name) {
            PENC_REQUIRE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name, " should be of the type of x or float32, however it is ",
                         t.scalar_type());
        };
        Tensor dense_gate, dense[4];
        if (gate.defined()) {
            own_or_float(gate, "gate");
            per_gate = rows_per_gate(x, gate, rows, channels);
            dense_gate = gate.detach().contiguous();
        }
        static constexpr const char* kNames[4] = {"post_weight", "post_bias", "pre_weight", "pre_bias"};
        const Tensor* first = nullptr;
        for (int i = 0; i < 4; ++i) {
            if (!params[i].defined()) continue;
            PENC_REQUIRE(i < 2 ? has_branch && o.post_norm : o.pre_norm, kNames[i], " is for a norm that is not asked for");
            PENC_REQUIRE(params[i].dim() == 1 && params[i].size(0) == channels, kNames[i], " should have a value for each of the ", channels,
                         " channels, however it has sizes ", params[i].sizes());
            own_or_float(params[i], kNames[i]);
            PENC_REQUIRE(first == nullptr || first->scalar_type() == params[i].scalar_type(), "weights and biases should be of one type");
            first = &params[i];
            dense[i] = params[i].detach().contiguous();
        }
        if (has_branch) y = at::empty(x.sizes(), x.options());
        if (o.pre_norm) n = at::empty(x.sizes(), x.options());
        if (rows != 0) {
            penc_norm a = norm_of(o, type, rows, channels, per_gate, dense_gate, dense);
            a.has_branch = has_branch;
            a.x = r.data(), a.x_stride = r.stride;
            if (has_branch) a.branch = b.data(), a.branch_stride = b.stride;
            if (differentiable && o.keep_8bit) {
                kept = room_for(x, rows, channels, has_branch ? 2 : 1);
                a.x_values = kept.q(), a.x_exponents = kept.e();
                if (has_branch) a.branch_values = kept.q(1), a.branch_exponents = kept.e(1);
            }
            check(api.residual_norm(&a, has_branch ? y.data_ptr() : nullptr, o.pre_norm ? n.data_ptr() : nullptr, current_stream(x.device())),
                  "residual_norm");
        }
    }
    if (!differentiable) return {y, n};
    auto node = make_node<NormNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, branch, gate, params[0], params[1], params[2], params[3]));
    node->options = o;
    node->type = type;
    node->rows = rows, node->channels = channels, node->per_gate = per_gate;
    node->has_branch = has_branch, node->has_y = has_branch;
    node->sizes = x.sizes().vec();
    for (int i = 0; i < 5; ++i) {
        const Tensor& p = i == 0 ? gate : params[i - 1];
        if (p.defined()) node->param_sizes[i] = p.sizes().vec(), node->param_types[i] = p.scalar_type();
    }
    const Tensor none;
    node->save({o.keep_8bit ? &none : &x, o.keep_8bit ? &none : &branch, &kept.bytes, &gate, &params[0], &params[1], &params[2], &params[3]});
    if (y.defined()) torch::autograd::set_history(y, node);
    if (n.defined()) torch::autograd::set_history(n, node);
    return {y, n};
}

// ------------------------------------------------------------------------------------------
// Python

Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }

// layers_keep(x) -> the checkpoint: int8, values and behind them exponents
PyObject* py_keep(PyObject*, PyObject* x_arg) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor& x = tensor_arg(x_arg, "x");
        require_plain({&x});
        Checkpoint kept;
        {
            NoGil no_gil;
            at::NoGradGuard no_grad;
            const c10::DeviceGuard device(x.device());
            kept = keep(x.detach(), "x");
        }
        return THPVariable_Wrap(std::move(kept.bytes));
    });
}

Checkpoint checkpoint_of(const Tensor& bytes, int64_t rows, int64_t channels) {
    require_plain({&bytes});
    PENC_REQUIRE(rows >= 0 && channels >= 1 && channels <= PENC_MAX_CHANNELS && bytes.scalar_type() == at::kChar && bytes.dim() == 1 && bytes.is_contiguous() &&
                     bytes.numel() == Checkpoint::size(rows, channels, 1),
                 "not a checkpoint of ", rows, " rows of ", channels, " channels");
    return {bytes, rows, channels};
}

// layers_restore(checkpoint, rows, channels, type) -> (rows, channels)
PyObject* py_restore(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 4, "layers_restore takes 4 arguments");
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor& bytes = tensor_arg(args[0], "checkpoint");
        const int64_t rows = PyLong_AsLongLong(args[1]), channels = PyLong_AsLongLong(args[2]);
        const long type = PyLong_AsLong(args[3]);
        if (PyErr_Occurred()) return nullptr;
        Tensor x;
        {
            NoGil no_gil;
            at::NoGradGuard no_grad;
            const Checkpoint kept = checkpoint_of(bytes, rows, channels);
            const c10::DeviceGuard device(bytes.device());
            x = at::empty({rows, channels}, bytes.options().dtype(scalar_type_of(type)));
            check(api.restore(static_cast<int>(type), rows, channels, kept.q(), kept.e(), x.data_ptr(), current_stream(x.device())), "unpack");
        }
        return THPVariable_Wrap(std::move(x));
    });
}

// layers_weight_grad(checkpoint, rows, channels, grad, bias, type) -> (weight gradient, bias gradient or None)
PyObject* py_weight_grad(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 6, "layers_weight_grad takes 6 arguments");
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor& bytes = tensor_arg(args[0], "checkpoint");
        const int64_t rows = PyLong_AsLongLong(args[1]), channels = PyLong_AsLongLong(args[2]);
        const Tensor& grad = tensor_arg(args[3], "grad");
        const int bias = PyObject_IsTrue(args[4]);
        const long type = PyLong_AsLong(args[5]);
        if (PyErr_Occurred()) return nullptr;
        std::pair<Tensor, Tensor> out;
        {
            NoGil no_gil;
            at::NoGradGuard no_grad;
            const Checkpoint kept = checkpoint_of(bytes, rows, channels);
            require_plain({&bytes, &grad});
            const c10::DeviceGuard device(grad.device());
            out = weight_grad(kept, channels, grad.detach(), scalar_type_of(type), bias != 0);
        }
        if (bias == 0) return Py_BuildValue("NO", THPVariable_Wrap(std::move(out.first)), Py_None);
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(out.first)), THPVariable_Wrap(std::move(out.second)));
    });
}

// layers_linear(x, weight, bias or None)
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 3, "layers_linear takes 3 arguments");
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight"), bias = optional_arg(args[2], "bias");
        Tensor y;
        {
            NoGil no_gil;
            y = linear(x, weight, bias);
        }
        return THPVariable_Wrap(std::move(y));
    });
}

// layers_activation(x, kind, gated, keep_8bit)
PyObject* py_activation(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 4, "layers_activation takes 4 arguments");
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor& x = tensor_arg(args[0], "x");
        const long kind = PyLong_AsLong(args[1]);
        const int gated = PyObject_IsTrue(args[2]), keep_8bit = PyObject_IsTrue(args[3]);
        if (PyErr_Occurred()) return nullptr;
        Tensor y;
        {
            NoGil no_gil;
            y = activation(x, static_cast<int>(kind), gated != 0, keep_8bit != 0);
        }
        return THPVariable_Wrap(std::move(y));
    });
}

// layers_residual_norm(x, branch, gate, post_weight, post_bias, pre_weight, pre_bias (each or None), residual_scale, post_norm, pre_norm, kind, eps,
//                      keep_8bit) -> (y or None, n or None)
PyObject* py_residual_norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 13, "layers_residual_norm takes 13 arguments");
        TORCH_CHECK(api.keep != nullptr, "bind() has not been called");
        const Tensor &x = tensor_arg(args[0], "x"), branch = optional_arg(args[1], "branch"), gate = optional_arg(args[2], "gate");
        const Tensor params[4] = {optional_arg(args[3], "post_weight"), optional_arg(args[4], "post_bias"), optional_arg(args[5], "pre_weight"),
                                  optional_arg(args[6], "pre_bias")};
        NormOptions o;
        PENC_REQUIRE(!THPVariable_Check(args[7]) && !THPVariable_Check(args[11]), "residual_scale and eps should be numbers: they have no gradient");
        o.scale = PyFloat_AsDouble(args[7]);
        o.post_norm = PyObject_IsTrue(args[8]) == 1, o.pre_norm = PyObject_IsTrue(args[9]) == 1;
        o.kind = static_cast<int>(PyLong_AsLong(args[10]));
        o.eps = PyFloat_AsDouble(args[11]);
        o.keep_8bit = PyObject_IsTrue(args[12]) == 1;
        if (PyErr_Occurred()) return nullptr;
        std::pair<Tensor, Tensor> out;
        {
            NoGil no_gil;
            out = residual_norm(x, branch, gate, params, o);
        }
        const auto wrapped = [](Tensor& t) {
            if (t.defined()) return THPVariable_Wrap(std::move(t));
            Py_INCREF(Py_None);
            return Py_None;
        };
        PyObject* const y = wrapped(out.first);
        return Py_BuildValue("NN", y, wrapped(out.second));
    });
}

template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name, const char* doc) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFunction)), METH_FASTCALL, doc};
}
PyMethodDef methods[] = {
    {"layers_keep", py_keep, METH_O, "a tensor in 8 bits"},
    fast<py_restore>("layers_restore", "the values that a checkpoint stands for"),
    fast<py_weight_grad>("layers_weight_grad", "a linear layer's weight and bias gradient from its kept input"),
    fast<py_linear>("layers_linear", "a linear layer that keeps its input in 8 bits"),
    fast<py_activation>("layers_activation", "an activation that keeps its input in 8 bits"),
    fast<py_residual_norm>("layers_residual_norm", "the norms around a residual, with its gate and scale"),
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace penc_torch {

void bind_layers(void* library) {
#define PENC_FN(fn)                                                           \
    api.fn = reinterpret_cast<decltype(api.fn)>(dlsym(library, "penc_" #fn)); \
    TORCH_CHECK(api.fn != nullptr, "the library does not export penc_" #fn)
    PENC_FN(status_string);
    PENC_FN(kept_pitch);
    PENC_FN(kept_blocks);
    PENC_FN(restore);
    PENC_FN(activation);
    PENC_FN(activation_backward);
    PENC_FN(weight_grad_workspace_bytes);
    PENC_FN(weight_grad);
    PENC_FN(residual_norm);
    PENC_FN(residual_norm_workspace_bytes);
    PENC_FN(residual_norm_backward);
    PENC_FN(keep);
#undef PENC_FN
}

bool add_layer_functions(PyObject* module) { return PyModule_AddFunctions(module, methods) == 0; }

}  // namespace penc_torch
