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
};

void require_matrices(const Tensor& t, const char* name) {
    type_of(t.scalar_type(), name);
    PENC_REQUIRE(t.dim() >= 2 && t.size(-1) >= 1 && t.size(-2) >= 1 && t.size(-1) <= PENC_MAX_MATRIX_SIDE && t.size(-2) <= PENC_MAX_MATRIX_SIDE, name,
                 " should be matrices (..., rows, columns) with sides of 1 to ", PENC_MAX_MATRIX_SIDE, ", however it has sizes ", t.sizes());
    PENC_REQUIRE(t.numel() / (t.size(-1) * t.size(-2)) <= PENC_MAX_MATRICES, name, " has more than ", PENC_MAX_MATRICES, " matrices");
}

void require_options(const Options& o) {
    PENC_REQUIRE(o.steps >= 1 && o.steps <= PENC_MAX_ORTHOGONAL_STEPS, "steps should be 1 to ", PENC_MAX_ORTHOGONAL_STEPS, ", however they are ", o.steps);
    PENC_REQUIRE(o.eps >= 1e-30 && o.eps < 1e30, "eps should be a positive number, however it is ", o.eps);
}

// The matrices of `update` (dense) into `result` (dense).
void orthogonalise(const Tensor& update, const Tensor& result, const Options& o) {
    const int64_t rows = update.size(-2), columns = update.size(-1);
    const penc_orthogonal matrices{type_of(update.scalar_type(), "update"), o.halves, update.numel() / (rows * columns), rows, columns, static_cast<int>(o.steps),
                                   static_cast<float>(o.a), static_cast<float>(o.b), static_cast<float>(o.c), static_cast<float>(o.eps)};
    const size_t n = api.orthogonal_workspace_bytes(&matrices);
    const Tensor ws = at::empty({static_cast<int64_t>(n)}, update.options().dtype(at::kByte));
    const int status = api.orthogonal_matrices(&matrices, update.const_data_ptr(), result.data_ptr(), ws.data_ptr(), n, current_stream(update.device()));
    PENC_REQUIRE(status != PENC_ERR_UNSUPPORTED_KIND, "coefficients should keep singular values under 3 and the factor under 15, however they are ", o.a, ", ", o.b, ", ", o.c);
    check(status, "orthogonalise");
}

Options options_of(PyObject* const* args) {
    Options o;
    o.steps = PyLong_AsLongLong(args[0]);
    o.a = PyFloat_AsDouble(args[1]), o.b = PyFloat_AsDouble(args[2]), o.c = PyFloat_AsDouble(args[3]), o.eps = PyFloat_AsDouble(args[4]);
    o.halves = PyObject_IsTrue(args[5]);
    return o;
}

// orthogonalise(update, steps, a, b, c, eps, halves)
PyObject* py_orthogonalise(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 7, "orthogonalise takes 7 arguments");
        TORCH_CHECK(api.orthogonal_matrices != nullptr, "bind() has not been called");
        const Tensor& update = tensor_arg(args[0], "update");
        const Options o = options_of(args + 1);
        if (PyErr_Occurred()) return nullptr;
        Tensor result;
        {
            NoGil no_gil;
            require_plain({&update});
            require_matrices(update, "update");
            require_options(o);
            at::NoGradGuard no_grad;
            const c10::DeviceGuard device(update.device());
            const Tensor dense = update.detach().contiguous();
            result = at::empty(update.sizes(), update.options());
            orthogonalise(dense, result, o);
        }
        return THPVariable_Wrap(std::move(result));
    });
}

constexpr int64_t kValuesAtOnce = int64_t{1} << 28;  // so that updates and workspaces stay within a few GB

void muon_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& averages, const Options& o, double momentum,
               int nesterov, double decay, double rate) {
    const Tensor& first = params[0];
    require_matrices(first, "a parameter");
    require_options(o);
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
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kValuesAtOnce / values, PENC_MAX_MATRICES / stack));
    const size_t size = first.element_size();
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

// muon_step(params, grads, averages, steps, a, b, c, eps, halves, momentum, nesterov, decay, rate): lists of dense tensors of one size, type and device
PyObject* py_muon_step(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        TORCH_CHECK(n_args == 13, "muon_step takes 13 arguments");
        TORCH_CHECK(api.orthogonal_matrices != nullptr, "bind() has not been called");
        std::vector<Tensor> lists[3];
        for (int k = 0; k < 3; ++k) {
            TORCH_CHECK(PyList_Check(args[k]) && PyList_Size(args[k]) == PyList_Size(args[0]), "muon_step takes three lists of one length");
            for (Py_ssize_t i = 0; i < PyList_Size(args[k]); ++i) lists[k].push_back(tensor_arg(PyList_GetItem(args[k], i), "a parameter, gradient or average"));
        }
        const Options o = options_of(args + 3);
        const double momentum = PyFloat_AsDouble(args[9]), decay = PyFloat_AsDouble(args[11]), rate = PyFloat_AsDouble(args[12]);
        const int nesterov = PyObject_IsTrue(args[10]);
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
