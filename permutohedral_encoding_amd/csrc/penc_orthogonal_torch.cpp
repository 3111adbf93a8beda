// Orthogonalised updates: what optim.py calls for them.
#include <dlfcn.h>

#include "penc_layers_torch.hpp"

namespace {

using namespace penc_torch;

struct Api {
#define PENC_FN(name) decltype(&penc_##name) name = nullptr
    PENC_FN(status_string);
    PENC_FN(orthogonal_workspace_bytes);
    PENC_FN(orthogonal_matrices);
    PENC_FN(muon_momentum);
    PENC_FN(muon_apply);
#undef PENC_FN
} api;

void check(int status, const char* what) {
    if (status != PENC_OK) TORCH_CHECK(false, what, ": ", api.status_string(status), " (status ", status, ")");
}

struct Options {
    int64_t steps;
    double a, b, c, eps;
    int halves;
    int64_t most_bytes;  // of a workspace, and of the updates of several parameters
};

void require_matrices(const Tensor& t, const char* name) {
    type_of(t.scalar_type(), name);
    PENC_REQUIRE(t.dim() >= 2 && t.size(-1) >= 1 && t.size(-2) >= 1 && t.size(-1) <= PENC_MAX_MATRIX_SIDE && t.size(-2) <= PENC_MAX_MATRIX_SIDE, name,
                 " should be matrices (..., rows, columns) with sides of 1 to ", PENC_MAX_MATRIX_SIDE, ", however it has sizes ", t.sizes());
    PENC_REQUIRE(t.numel() / (t.size(-1) * t.size(-2)) <= PENC_MAX_MATRICES, name, " has more than ", PENC_MAX_MATRICES, " matrices");
}

void require_options(const Options& o) {
    PENC_REQUIRE(o.steps >= 1 && o.steps <= PENC_MAX_ORTHOGONAL_STEPS, "steps should be 1 to ", PENC_MAX_ORTHOGONAL_STEPS, ", however they are ", o.steps);
    PENC_REQUIRE(o.most_bytes >= 0, "a workspace should have no negative number of bytes, however it has ", o.most_bytes);
    PENC_REQUIRE(o.eps >= 1e-30 && o.eps < 1e30, "eps should be a positive number, however it is ", o.eps);
}

// The matrices of `update` (dense) into `result` (dense): as many at a time as the workspace has room for, and one, or two or four of them that together are
// whole fours of values, at least.
void orthogonalise(const Tensor& update, const Tensor& result, const Options& o) {
    const int64_t rows = update.size(-2), columns = update.size(-1), values = rows * columns, all = update.numel() / values;
    const int64_t fours = values % 4 == 0 ? 1 : values % 2 == 0 ? 2 : 4;
    penc_orthogonal matrices{type_of(update.scalar_type(), "update"), o.halves, all, rows, columns, static_cast<int>(o.steps),
                             static_cast<float>(o.a), static_cast<float>(o.b), static_cast<float>(o.c), static_cast<float>(o.eps)};
    while (matrices.matrices > fours && api.orthogonal_workspace_bytes(&matrices) > static_cast<size_t>(o.most_bytes))
        matrices.matrices = (matrices.matrices / 2 + fours - 1) / fours * fours;
    const int64_t most = std::max<int64_t>(matrices.matrices, 1), bytes = values * static_cast<int64_t>(update.element_size());
    for (int64_t first = 0; first < all; first += most) {
        matrices.matrices = std::min(most, all - first);
        const size_t n = api.orthogonal_workspace_bytes(&matrices);
        const Tensor ws = at::empty({static_cast<int64_t>(n)}, update.options().dtype(at::kByte));
        check(api.orthogonal_matrices(&matrices, static_cast<const char*>(update.const_data_ptr()) + first * bytes,
            static_cast<char*>(result.data_ptr()) + first * bytes, ws.data_ptr(), n,
                                      current_stream(update.device())),
              "orthogonalise");
    }
}

// Refuses coefficients and eps before anything is changed.
void require_accepted(const Options& o) {
    require_options(o);
    const penc_orthogonal none{PENC_FP32, 0, 0, 1, 1, static_cast<int>(o.steps), static_cast<float>(o.a), static_cast<float>(o.b),
        static_cast<float>(o.c), static_cast<float>(o.eps)};
    const int status = api.orthogonal_matrices(&none, nullptr, nullptr, nullptr, 0, nullptr);
    PENC_REQUIRE(status != PENC_ERR_UNSUPPORTED_KIND, "coefficients should keep singular values under 3 and the factor under 15, however they are ",
        o.a, ", ", o.b, ", ", o.c);
    check(status, "orthogonalise");
}

Options options_of(PyObject* const* args) {
    Options o;
    o.steps = PyLong_AsLongLong(args[0]);
    o.a = PyFloat_AsDouble(args[1]), o.b = PyFloat_AsDouble(args[2]), o.c = PyFloat_AsDouble(args[3]), o.eps = PyFloat_AsDouble(args[4]);
    o.halves = PyObject_IsTrue(args[5]);
    o.most_bytes = PyLong_AsLongLong(args[6]);
    return o;
}

// orthogonalise(update, steps, a, b, c, eps, halves, most_bytes)
PyObject* py_orthogonalise(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 8, "orthogonalise takes 8 arguments");
        TORCH_CHECK(api.orthogonal_matrices != nullptr, "bind() has not been called");
        const Tensor& update = tensor_arg(args[0], "update");
        const Options o = options_of(args + 1);
        if (PyErr_Occurred()) return nullptr;
        Tensor result;
        {
            NoGil no_gil;
            require_plain({&update});
            require_matrices(update, "update");
            require_accepted(o);
            at::NoGradGuard no_grad;
            const c10::DeviceGuard device(update.device());
            const Tensor dense = update.detach().contiguous();
            result = at::empty(update.sizes(), update.options());
            orthogonalise(dense, result, o);
        }
        return THPVariable_Wrap(std::move(result));
    });
}

// orthogonal_options(steps, a, b, c, eps, halves, most_bytes): raises what the functions here would
PyObject* py_orthogonal_options(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 7, "orthogonal_options takes 7 arguments");
        TORCH_CHECK(api.orthogonal_matrices != nullptr, "bind() has not been called");
        const Options o = options_of(args);
        if (PyErr_Occurred()) return nullptr;
        require_accepted(o);
        Py_RETURN_NONE;
    });
}

// orthogonal_sizes(param, grad), likewise
PyObject* py_orthogonal_sizes(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 2, "orthogonal_sizes takes 2 arguments");
        const Tensor &param = tensor_arg(args[0], "a parameter"), &grad = tensor_arg(args[1], "a gradient");
        require_plain({&param, &grad});
        require_matrices(param, "a parameter");
        Py_RETURN_NONE;
    });
}

void muon_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& averages, const Options& o, double momentum,
               int nesterov, double decay, double rate) {
    const Tensor& first = params[0];
    require_matrices(first, "a parameter");
    require_accepted(o);
    for (size_t i = 0; i < params.size(); ++i) {
        require_plain({&params[i], &grads[i], &averages[i]});
        TORCH_CHECK(params[i].sizes() == first.sizes() && params[i].scalar_type() == first.scalar_type() && params[i].device() == first.device() &&
                        grads[i].sizes() == first.sizes() && grads[i].scalar_type() == first.scalar_type() && grads[i].device() == first.device() &&
                        averages[i].sizes() == first.sizes() && averages[i].scalar_type() == at::kFloat && averages[i].device() == first.device() &&
                        params[i].is_contiguous() && grads[i].is_contiguous() && averages[i].is_contiguous(),
                    "Muon: parameters, gradients and averages must be contiguous, of one size, type and device");
    }
    at::NoGradGuard no_grad;
    const c10::DeviceGuard device(first.device());
    void* const stream = current_stream(first.device());
    const int type = type_of(first.scalar_type(), "a parameter");
    const int64_t values = first.numel(), stack = values / (first.size(-1) * first.size(-2));
    if (values == 0) return;
    const int64_t size = static_cast<int64_t>(first.element_size());
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(o.most_bytes / (2 * size * values), PENC_MAX_MATRICES / stack));
    for (int64_t begin = 0; begin < static_cast<int64_t>(params.size()); begin += most) {
        const int64_t count = std::min<int64_t>(most, static_cast<int64_t>(params.size()) - begin);
        const Tensor update = at::empty({count * stack, first.size(-2), first.size(-1)}, first.options()), result = at::empty_like(update);
        for (int64_t i = 0; i < count; ++i)
            check(api.muon_momentum(type, values, grads[begin + i].const_data_ptr(), static_cast<float*>(averages[begin + i].data_ptr()),
                                    static_cast<float>(momentum), nesterov, static_cast<char*>(update.data_ptr()) + i * values * size, stream),
                  "Muon");
        orthogonalise(update, result, o);
        for (int64_t i = 0; i < count; ++i) {
            check(api.muon_apply(type, values, params[begin + i].data_ptr(), static_cast<const char*>(result.const_data_ptr()) + i * values * size,
                                 static_cast<float>(decay), static_cast<float>(rate), stream),
                  "Muon");
            params[begin + i].unsafeGetTensorImpl()->bump_version();
        }
    }
}

// muon_step(params, grads, averages, steps, a, b, c, eps, halves, most_bytes, momentum, nesterov, decay, rate): lists of dense tensors of one size, type and
// device
PyObject* py_muon_step(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 14, "muon_step takes 14 arguments");
        TORCH_CHECK(api.orthogonal_matrices != nullptr, "bind() has not been called");
        std::vector<Tensor> lists[3];
        for (int k = 0; k < 3; ++k) {
            TORCH_CHECK(PyList_Check(args[k]) && PyList_Size(args[k]) == PyList_Size(args[0]), "muon_step takes three lists of one length");
            for (Py_ssize_t i = 0; i < PyList_Size(args[k]); ++i) lists[k].push_back(tensor_arg(PyList_GetItem(args[k], i), "a parameter, gradient or average"));
        }
        const Options o = options_of(args + 3);
        const double momentum = PyFloat_AsDouble(args[10]), decay = PyFloat_AsDouble(args[12]), rate = PyFloat_AsDouble(args[13]);
        const int nesterov = PyObject_IsTrue(args[11]);
        if (PyErr_Occurred()) return nullptr;
        const auto& [params, grads, averages] = lists;
        if (params.empty()) Py_RETURN_NONE;
        {
            NoGil no_gil;
            muon_step(params, grads, averages, o, momentum, nesterov, decay, rate);
        }
        Py_RETURN_NONE;
    });
}
PyMethodDef methods[] = {fast<py_orthogonalise>("orthogonalise", "nearly orthogonal matrices from updates"),
                         fast<py_orthogonal_options>("orthogonal_options", "what steps, coefficients and eps are refused for"),
                         fast<py_orthogonal_sizes>("orthogonal_sizes", "what a parameter and its gradient are refused for"),
                         fast<py_muon_step>("muon_step", "a step with orthogonalised updates"),
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

namespace penc_torch {

void bind_orthogonal(void* library) {
#define PENC_FN(fn)                                                           \
    api.fn = reinterpret_cast<decltype(api.fn)>(dlsym(library, "penc_" #fn)); \
    TORCH_CHECK(api.fn != nullptr, "the library does not export penc_" #fn)
    PENC_FN(status_string);
    PENC_FN(orthogonal_workspace_bytes);
    PENC_FN(muon_momentum);
    PENC_FN(muon_apply);
    PENC_FN(orthogonal_matrices);
#undef PENC_FN
}

bool add_orthogonal_functions(PyObject* module) { return PyModule_AddFunctions(module, methods) == 0; }

}  // namespace penc_torch
