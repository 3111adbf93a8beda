// Rows that go to experts: the functions of layers.py for them, through autograd to the kernels and back.
#include <dlfcn.h>

#include "penc_layers_torch.hpp"

namespace {

using namespace penc_torch;

struct Api {
#define PENC_FN(name) decltype(&penc_##name) name = nullptr
    PENC_FN(status_string);
    PENC_FN(route);
    PENC_FN(route_backward);
    PENC_FN(plan);
    PENC_FN(plan_workspace_bytes);
    PENC_FN(dispatch);
    PENC_FN(combine);
    PENC_FN(combine_backward);
    PENC_FN(expert_linear);
    PENC_FN(expert_linear_input_grad);
    PENC_FN(expert_weight_grad_workspace_bytes);
    PENC_FN(expert_linear_grads);
    PENC_FN(expert_bias_grad_workspace_bytes);
    PENC_FN(expert_bias_grad);
#undef PENC_FN
} api;

void check(int status, const char* what) {
    if (status != PENC_OK) TORCH_CHECK(false, what, ": ", api.status_string(status), " (status ", status, ")");
}

// ------------------------------------------------------------------------------------------
// plans

// Where the choices (..., k) of rows stand when they are sorted by expert.
struct Plan {
    Tensor positions, offsets;  // int32 (..., k) and (experts + 1,)
    int64_t rows = 0, choices = 0;
    int experts = 0;

    const int32_t* at() const { return static_cast<const int32_t*>(positions.const_data_ptr()); }
    const int32_t* begins() const { return static_cast<const int32_t*>(offsets.const_data_ptr()); }
    const int32_t* routed() const { return begins() + experts; }
};

void require_experts(int64_t experts) {
    PENC_REQUIRE(experts >= 1 && experts <= PENC_MAX_EXPERTS, "there should be 1 to ", PENC_MAX_EXPERTS, " experts, however there are ", experts);
}

Plan plan_of(const Tensor& positions, const Tensor& offsets) {
    require_plain({&positions, &offsets});
    PENC_REQUIRE(positions.scalar_type() == at::kInt && positions.dim() >= 1 && positions.is_contiguous() && offsets.scalar_type() == at::kInt &&
                     offsets.dim() == 1 && offsets.is_contiguous() && positions.size(-1) >= 1 && positions.size(-1) <= PENC_MAX_CHOICES && offsets.size(0) >= 2,
                 "a routing should be as routing() or route() make it");
    require_experts(offsets.size(0) - 1);
    Plan p{positions, offsets, 0, positions.size(-1), static_cast<int>(offsets.size(0) - 1)};
    p.rows = positions.numel() / p.choices;
    return p;
}

// -> positions and offsets of chosen experts (..., k), int32 or int64
Plan make_plan(const Tensor& chosen, int64_t experts) {
    PENC_REQUIRE(chosen.scalar_type() == at::kInt || chosen.scalar_type() == at::kLong, "experts should be of type int32 or int64, however they are ",
                 chosen.scalar_type());
    PENC_REQUIRE(chosen.dim() >= 1 && chosen.size(-1) >= 1 && chosen.size(-1) <= PENC_MAX_CHOICES, "each row should have 1 to ", PENC_MAX_CHOICES,
                 " experts, however experts have sizes ", chosen.sizes());
    require_experts(experts);
    const Tensor dense = chosen.contiguous();
    const auto options = chosen.options().dtype(at::kInt);
    Plan p{at::empty(chosen.sizes(), options), at::empty({experts + 1}, options), chosen.numel() / chosen.size(-1), chosen.size(-1), static_cast<int>(experts)};
    const size_t n = api.plan_workspace_bytes(chosen.numel(), p.experts);
    const Tensor ws = at::empty({static_cast<int64_t>(n)}, chosen.options().dtype(at::kByte));
    check(api.plan(chosen.scalar_type() == at::kInt ? 4 : 8, chosen.numel(), p.experts, dense.const_data_ptr(), static_cast<int32_t*>(p.positions.data_ptr()),
                   static_cast<int32_t*>(p.offsets.data_ptr()), ws.data_ptr(), n, current_stream(chosen.device())),
          "routing");
    return p;
}

// Nodes of sums in full precision.
struct ExpertNode : public LayerNode {
    const char* why_once() const override { return "no rule for that is there"; }
};

Plan saved_plan(const Tensor& positions, const Tensor& offsets, int64_t rows, int64_t choices, int experts) {
    TORCH_CHECK(positions.defined() && offsets.defined() && positions.is_cuda() && offsets.is_cuda() && positions.scalar_type() == at::kInt &&
                    offsets.scalar_type() == at::kInt && positions.is_contiguous() && offsets.is_contiguous() && positions.numel() == rows * choices &&
                    offsets.numel() == experts + 1,
                "a routing saved for the backward has come back in another form");
    return {positions, offsets, rows, choices, experts};
}

// ------------------------------------------------------------------------------------------
// route

struct RouteNode : public ExpertNode {
    bool normalise = true;
    int type = 0;
    int64_t rows = 0, choices = 0;
    std::vector<int64_t> sizes, weight_sizes;

    std::string name() const override { return "LayersRouteBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();  // logits (not with normalise), weights, chosen
        variable_list out(1);
        const Tensor& g = grads[0];
        const c10::DeviceGuard device(g.device());
        out[0] = at::empty(sizes, g.options().dtype(scalar_type_of(type)));
        if (rows == 0) return out;
        Rows logits;
        if (!normalise) {
            require_saved(t[0], sizes, scalar_type_of(type));
            logits = rows_of(t[0], "logits");
        }
        require_saved(t[1], weight_sizes, at::kFloat);
        require_saved(t[2], weight_sizes, at::kInt);
        const Tensor weights = t[1].contiguous(), chosen = t[2].contiguous(), grad = g.detach().to(at::kFloat).contiguous();
        check(api.route_backward(type, rows, static_cast<int>(sizes.back()), static_cast<int>(choices), normalise, normalise ? nullptr : logits.data(),
                                 logits.stride, static_cast<const float*>(weights.const_data_ptr()), static_cast<const int32_t*>(chosen.const_data_ptr()),
                                 static_cast<const float*>(grad.const_data_ptr()), out[0].data_ptr(), current_stream(g.device())),
              "route");
        return out;
    }
};

struct Routed {
    Tensor weights, chosen;
    Plan plan;
};

Routed route(const Tensor& logits, int64_t choices, bool normalise) {
    require_plain({&logits});
    const int type = type_of(logits.scalar_type(), "logits");
    const c10::DeviceGuard device(logits.device());
    const bool differentiable = any_requires_grad({&logits});
    Routed out;
    Rows r;
    std::vector<int64_t> sizes;
    {
        at::NoGradGuard no_grad;
        r = rows_of(logits.detach(), "logits");
        require_experts(r.channels);
        PENC_REQUIRE(choices >= 1 && choices <= r.channels && choices <= PENC_MAX_ROUTED, "a row should choose 1 to ", PENC_MAX_ROUTED, " of its ", r.channels,
                     " experts, however it chooses ", choices);
        sizes = logits.sizes().vec();
        sizes.back() = choices;
        out.weights = at::empty(sizes, logits.options().dtype(at::kFloat));
        out.chosen = at::empty(sizes, logits.options().dtype(at::kInt));
        check(api.route(type, r.n, static_cast<int>(r.channels), static_cast<int>(choices), normalise, r.data(), r.stride,
                        static_cast<float*>(out.weights.data_ptr()), static_cast<int32_t*>(out.chosen.data_ptr()), current_stream(logits.device())),
              "route");
        out.plan = make_plan(out.chosen, r.channels);
    }
    if (!differentiable) return out;
    auto node = make_node<RouteNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->normalise = normalise, node->type = type, node->rows = r.n, node->choices = choices;
    node->sizes = logits.sizes().vec(), node->weight_sizes = sizes;
    const Tensor none, weights = out.weights.detach();  // (the same values, and no cycle through the node)
    node->save({normalise ? &none : &logits, &weights, &out.chosen});
    torch::autograd::set_history(out.weights, node);
    return out;
}

// ------------------------------------------------------------------------------------------
// dispatch

struct DispatchNode : public ExpertNode {
    int type = 0, experts = 0;
    int64_t rows = 0, choices = 0;
    std::vector<int64_t> sizes;  // of x

    std::string name() const override { return "LayersDispatchBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();
        const c10::DeviceGuard device(grads[0].device());
        variable_list out(1);
        out[0] = at::empty(sizes, grads[0].options().dtype(scalar_type_of(type)));
        if (rows == 0) return out;
        const Plan plan = saved_plan(t[0], t[1], rows, choices, experts);
        const Rows g = grad_rows(grads[0], scalar_type_of(type));
        check(api.combine(type, type, rows, static_cast<int>(choices), sizes.back(), g.data(), g.stride, nullptr, plan.at(), plan.routed(), out[0].data_ptr(),
                          current_stream(out[0].device())),
              "dispatch");
        return out;
    }
};

// The rows (..., C) that the plan is of.
Rows planned_rows(const Tensor& x, const Plan& plan, const char* name) {
    const Rows r = rows_of(x, name);
    PENC_REQUIRE(x.sizes().slice(0, x.dim() - 1) == plan.positions.sizes().slice(0, plan.positions.dim() - 1), name, " should have the rows that were routed, ",
                 plan.positions.sizes().slice(0, plan.positions.dim() - 1), ", however it has sizes ", x.sizes());
    PENC_REQUIRE(r.channels <= PENC_MAX_CHANNELS, name, " has more than ", PENC_MAX_CHANNELS, " channels");
    return r;
}
// Rows (rows * k, C) sorted by expert.
Rows sorted_rows(const Tensor& y, const Plan& plan, const char* name) {
    PENC_REQUIRE(y.dim() == 2 && y.size(0) == plan.positions.numel(), name, " should have a row for each of the ", plan.positions.numel(),
                 " choices, however it has sizes ", y.sizes());
    const Rows r = rows_of(y, name);
    PENC_REQUIRE(r.channels <= PENC_MAX_CHANNELS, name, " has more than ", PENC_MAX_CHANNELS, " channels");
    return r;
}

Tensor dispatch(const Tensor& x, const Tensor& positions, const Tensor& offsets) {
    require_plain({&x, &positions, &offsets});
    const Plan plan = plan_of(positions, offsets);
    const int type = type_of(x.scalar_type(), "x");
    const c10::DeviceGuard device(x.device());
    const bool differentiable = any_requires_grad({&x});
    Tensor sorted;
    {
        at::NoGradGuard no_grad;
        const Rows r = planned_rows(x.detach(), plan, "x");
        sorted = at::empty({positions.numel(), r.channels}, x.options());
        check(api.dispatch(type, r.n, static_cast<int>(plan.choices), r.channels, r.data(), r.stride, plan.at(), plan.routed(), sorted.data_ptr(),
                           current_stream(x.device())),
              "dispatch");
    }
    if (!differentiable) return sorted;
    auto node = make_node<DispatchNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->type = type, node->experts = plan.experts, node->rows = plan.rows, node->choices = plan.choices;
    node->sizes = x.sizes().vec();
    node->save({&positions, &offsets});
    torch::autograd::set_history(sorted, node);
    return sorted;
}

// ------------------------------------------------------------------------------------------
// combine

struct CombineNode : public ExpertNode {
    int type = 0, weight_type = 0, experts = 0;
    int64_t rows = 0, choices = 0;
    std::vector<int64_t> sizes, weight_sizes;  // of y and of the weights

    std::string name() const override { return "LayersCombineBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();  // y (where the weights want a gradient), weights, positions, offsets
        const c10::DeviceGuard device(grads[0].device());
        const bool want_y = task_should_compute_output(0), want_weights = t[0].defined() && task_should_compute_output(1);
        variable_list out(2);
        const auto options = grads[0].options();
        if (want_y) out[0] = at::empty(sizes, options.dtype(scalar_type_of(type)));
        if (want_weights) out[1] = at::empty(weight_sizes, options.dtype(scalar_type_of(weight_type)));
        if (rows == 0) return out;
        const Plan plan = saved_plan(t[2], t[3], rows, choices, experts);
        require_saved(t[1], weight_sizes, scalar_type_of(weight_type));
        const Tensor weights = t[1].contiguous();
        Rows y;
        if (want_weights) {
            require_saved(t[0], sizes, scalar_type_of(type));
            y = rows_of(t[0], "y");
        }
        const Rows g = grad_rows(grads[0], scalar_type_of(type));
        check(api.combine_backward(type, weight_type, rows, static_cast<int>(choices), sizes.back(), g.data(), g.stride, want_weights ? y.data() : nullptr, y.stride,
                                   weights.const_data_ptr(), plan.at(), plan.routed(), want_y ? out[0].data_ptr() : nullptr,
                                   want_weights ? out[1].data_ptr() : nullptr, current_stream(grads[0].device())),
              "combine");
        return out;
    }
};

Tensor combine(const Tensor& y, const Tensor& weights, const Tensor& positions, const Tensor& offsets) {
    require_plain({&y, &weights, &positions, &offsets});
    const Plan plan = plan_of(positions, offsets);
    const int type = type_of(y.scalar_type(), "y"), weight_type = type_of(weights.scalar_type(), "weights");
    PENC_REQUIRE(weight_type == type || weight_type == PENC_FP32, "weights should be of the type of y or float32, however they are ", weights.scalar_type());
    PENC_REQUIRE(weights.sizes() == positions.sizes(), "weights should have a value for each choice, ", positions.sizes(), ", however they have sizes ",
                 weights.sizes());
    const c10::DeviceGuard device(y.device());
    const bool differentiable = any_requires_grad({&y, &weights});
    Tensor out;
    {
        at::NoGradGuard no_grad;
        const Rows r = sorted_rows(y.detach(), plan, "y");
        const Tensor dense = weights.detach().contiguous();
        std::vector<int64_t> sizes = positions.sizes().vec();
        sizes.back() = r.channels;
        out = at::empty(sizes, y.options());
        check(api.combine(type, weight_type, plan.rows, static_cast<int>(plan.choices), r.channels, r.data(), r.stride, dense.const_data_ptr(), plan.at(),
                          plan.routed(), out.data_ptr(), current_stream(y.device())),
              "combine");
    }
    if (!differentiable) return out;
    auto node = make_node<CombineNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(y, weights));
    node->type = type, node->weight_type = weight_type, node->experts = plan.experts, node->rows = plan.rows, node->choices = plan.choices;
    node->sizes = y.sizes().vec(), node->weight_sizes = weights.sizes().vec();
    const Tensor none;
    node->save({weights.requires_grad() ? &y : &none, &weights, &positions, &offsets});
    torch::autograd::set_history(out, node);
    return out;
}

// ------------------------------------------------------------------------------------------
// expert_linear

// Rows as the products read them: none overlaps another, and none is further from it than a tile's offsets reach.
Rows product_rows(Rows r) {
    if (r.n > 1 && (r.stride < r.channels || r.stride > PENC_MAX_EXPERT_STRIDE)) {
        r.values = r.values.clone(at::MemoryFormat::Contiguous);
        r.stride = r.channels;
    }
    return r;
}

struct ExpertLinearNode : public ExpertNode {
    int type = 0, experts = 0;
    int64_t rows = 0;
    std::vector<int64_t> sizes, weight_sizes;
    bool has_bias = false;

    std::string name() const override { return "LayersExpertLinearBackward"; }
    variable_list gradients(const variable_list& grads) override {
        const std::vector<Tensor> t = unpacked();  // x (where the weight wants a gradient), weight (where x does), offsets
        const auto scalar = scalar_type_of(type);
        const c10::DeviceGuard device(grads[0].device());
        TORCH_CHECK(t[2].defined() && t[2].is_cuda() && t[2].scalar_type() == at::kInt && t[2].is_contiguous() && t[2].numel() == experts + 1,
                    "a routing saved for the backward has come back in another form");
        const int32_t* const offsets = static_cast<const int32_t*>(t[2].const_data_ptr());
        const int64_t outputs = weight_sizes[1], channels = weight_sizes[2];
        const Rows g = product_rows(grad_rows(grads[0], scalar));
        const auto options = grads[0].options().dtype(scalar);
        void* const stream = current_stream(grads[0].device());
        variable_list out(3);
        const bool want_x = t[1].defined() && task_should_compute_output(0), want_bias = has_bias && task_should_compute_output(2);
        Tensor weight;
        if (want_x) {
            require_saved(t[1], weight_sizes, scalar);
            weight = t[1].contiguous();
            out[0] = at::empty(sizes, options);
        }
        if (want_bias) out[2] = at::empty({weight_sizes[0], outputs}, options);
        if (!t[0].defined() || !task_should_compute_output(1)) {
            if (want_x)
                check(api.expert_linear_input_grad(type, rows, experts, channels, outputs, g.data(), g.stride, weight.const_data_ptr(), offsets,
                    out[0].data_ptr(), stream),
                      "expert_linear");
            if (want_bias) {
                const size_t n = api.expert_bias_grad_workspace_bytes(type, rows, experts, outputs);
                const Tensor ws = at::empty({static_cast<int64_t>(n)}, options.dtype(at::kByte));
                check(api.expert_bias_grad(type, rows, experts, outputs, g.data(), g.stride, offsets, out[2].data_ptr(), ws.data_ptr(), n, stream), "expert_linear");
            }
            return out;
        }
        require_saved(t[0], sizes, scalar);
        const Rows x = product_rows(rows_of(t[0], "x"));
        out[1] = at::empty(weight_sizes, options);
        const size_t n = api.expert_weight_grad_workspace_bytes(type, rows, experts, channels, outputs);
        const Tensor ws = at::empty({static_cast<int64_t>(n)}, options.dtype(at::kByte));
        check(api.expert_linear_grads(type, rows, experts, channels, outputs, x.data(), x.stride, g.data(), g.stride, want_x ? weight.const_data_ptr() : nullptr, offsets,
                                      want_x ? out[0].data_ptr() : nullptr, out[1].data_ptr(), want_bias ? out[2].data_ptr() : nullptr, ws.data_ptr(), n, stream),
              "expert_linear");
        return out;
    }
};

Tensor expert_linear(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& positions, const Tensor& offsets) {
    require_plain({&x, &weight, &bias, &positions, &offsets});
    const Plan plan = plan_of(positions, offsets);
    const int type = type_of(x.scalar_type(), "x");
    PENC_REQUIRE(weight.scalar_type() == x.scalar_type() && (!bias.defined() || bias.scalar_type() == x.scalar_type()),
                 "x, weight and bias of expert_linear should be of one type");
    PENC_REQUIRE(weight.dim() == 3 && weight.size(0) == plan.experts && weight.size(1) >= 1 && weight.size(2) >= 1, "weight should have sizes (", plan.experts,
                 ", outputs, channels), however they are ", weight.sizes());
    const int64_t outputs = weight.size(1), channels = weight.size(2);
    PENC_REQUIRE(x.dim() == 2 && x.size(1) == channels, "expert_linear should have rows of ", channels, " channels, however x has sizes ", x.sizes());
    PENC_REQUIRE(outputs <= PENC_MAX_EXPERT_CHANNELS && channels <= PENC_MAX_EXPERT_CHANNELS, "an expert should have at most ", PENC_MAX_EXPERT_CHANNELS,
                 " channels and outputs");
    PENC_REQUIRE(!bias.defined() || (bias.dim() == 2 && bias.size(0) == plan.experts && bias.size(1) == outputs),
                 "expert_linear should have a bias for each expert and output");
    const c10::DeviceGuard device(x.device());
    const bool differentiable = any_requires_grad({&x, &weight, &bias});
    Tensor y;
    {
        at::NoGradGuard no_grad;
        const Rows r = product_rows(sorted_rows(x.detach(), plan, "x"));
        const Tensor w = weight.detach().contiguous(), b = bias.defined() ? bias.detach().contiguous() : Tensor();
        y = at::empty({x.size(0), outputs}, x.options());
        check(api.expert_linear(type, r.n, plan.experts, channels, outputs, r.data(), r.stride, w.const_data_ptr(), b.defined() ? b.const_data_ptr() : nullptr,
                                plan.begins(), y.data_ptr(), current_stream(x.device())),
              "expert_linear");
    }
    if (!differentiable) return y;
    auto node = make_node<ExpertLinearNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->type = type, node->experts = plan.experts, node->rows = x.size(0);
    node->sizes = x.sizes().vec(), node->weight_sizes = weight.sizes().vec();
    node->has_bias = bias.defined();
    const Tensor none;
    node->save({weight.requires_grad() ? &x : &none, x.requires_grad() ? &weight : &none, &offsets});
    torch::autograd::set_history(y, node);
    return y;
}

// ------------------------------------------------------------------------------------------
// Python

void require_bound() { TORCH_CHECK(api.route != nullptr, "bind() has not been called"); }

// layers_route(logits, choices, normalise) -> (weights, experts, positions, offsets)
PyObject* py_route(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 3, "layers_route takes 3 arguments");
        require_bound();
        const Tensor& logits = tensor_arg(args[0], "logits");
        const int64_t choices = PyLong_AsLongLong(args[1]);
        const int normalise = PyObject_IsTrue(args[2]);
        if (PyErr_Occurred()) return nullptr;
        Routed r;
        {
            NoGil no_gil;
            r = route(logits, choices, normalise != 0);
        }
        return Py_BuildValue("NNNN", THPVariable_Wrap(std::move(r.weights)), THPVariable_Wrap(std::move(r.chosen)), THPVariable_Wrap(std::move(r.plan.positions)),
                             THPVariable_Wrap(std::move(r.plan.offsets)));
    });
}

// layers_plan(experts, number) -> (positions, offsets)
PyObject* py_plan(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 2, "layers_plan takes 2 arguments");
        require_bound();
        const Tensor& chosen = tensor_arg(args[0], "experts");
        const int64_t experts = PyLong_AsLongLong(args[1]);
        if (PyErr_Occurred()) return nullptr;
        Plan p;
        {
            NoGil no_gil;
            require_plain({&chosen});
            at::NoGradGuard no_grad;
            const c10::DeviceGuard device(chosen.device());
            p = make_plan(chosen, experts);
        }
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(p.positions)), THPVariable_Wrap(std::move(p.offsets)));
    });
}

// layers_dispatch(x, positions, offsets)
PyObject* py_dispatch(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 3, "layers_dispatch takes 3 arguments");
        require_bound();
        const Tensor &x = tensor_arg(args[0], "x"), &positions = tensor_arg(args[1], "positions"), &offsets = tensor_arg(args[2], "offsets");
        Tensor out;
        {
            NoGil no_gil;
            out = dispatch(x, positions, offsets);
        }
        return THPVariable_Wrap(std::move(out));
    });
}

// layers_combine(y, weights, positions, offsets)
PyObject* py_combine(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 4, "layers_combine takes 4 arguments");
        require_bound();
        const Tensor &y = tensor_arg(args[0], "y"), &weights = tensor_arg(args[1], "weights"), &positions = tensor_arg(args[2], "positions"),
                     &offsets = tensor_arg(args[3], "offsets");
        Tensor out;
        {
            NoGil no_gil;
            out = combine(y, weights, positions, offsets);
        }
        return THPVariable_Wrap(std::move(out));
    });
}

// layers_expert_linear(x, weight, bias or None, positions, offsets)
PyObject* py_expert_linear(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 5, "layers_expert_linear takes 5 arguments");
        require_bound();
        const Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight"), bias = optional_arg(args[2], "bias"),
                     &positions = tensor_arg(args[3], "positions"), &offsets = tensor_arg(args[4], "offsets");
        Tensor out;
        {
            NoGil no_gil;
            out = expert_linear(x, weight, bias, positions, offsets);
        }
        return THPVariable_Wrap(std::move(out));
    });
}

PyMethodDef methods[] = {fast<py_route>("layers_route", "the experts of rows, their weights, and where the choices stand when they are sorted by expert"),
                         fast<py_plan>("layers_plan", "where given choices stand"),
                         fast<py_dispatch>("layers_dispatch", "rows sorted by expert"),
                         fast<py_combine>("layers_combine", "weighted sums of sorted rows"),
                         fast<py_expert_linear>("layers_expert_linear", "a linear layer of each expert on its own rows"),
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace penc_torch {

void bind_experts(void* library) {
#define PENC_FN(fn)                                                           \
    api.fn = reinterpret_cast<decltype(api.fn)>(dlsym(library, "penc_" #fn)); \
    TORCH_CHECK(api.fn != nullptr, "the library does not export penc_" #fn)
    PENC_FN(status_string);
    PENC_FN(route_backward);
    PENC_FN(plan);
    PENC_FN(plan_workspace_bytes);
    PENC_FN(dispatch);
    PENC_FN(combine);
    PENC_FN(combine_backward);
    PENC_FN(expert_linear);
    PENC_FN(expert_linear_input_grad);
    PENC_FN(expert_weight_grad_workspace_bytes);
    PENC_FN(expert_linear_grads);
    PENC_FN(expert_bias_grad_workspace_bytes);
    PENC_FN(expert_bias_grad);
    PENC_FN(route);
#undef PENC_FN
}

bool add_expert_functions(PyObject* module) { return PyModule_AddFunctions(module, methods) == 0; }

}  // namespace penc_torch
