// What the sources of the extension _penc_torch share: checks, the current stream, exceptions on their way into Python.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <utility>

namespace penc_torch {

using at::Tensor;

// penc_layers_torch.cpp: takes its entry points from the library; adds its functions to the module.
void bind_layers(void* library);
bool add_layer_functions(PyObject* module);

#define PENC_REQUIRE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

inline void* current_stream(const at::Device& device) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream();
}

inline const Tensor& tensor_arg(PyObject* o, const char* name) {
    PENC_REQUIRE(THPVariable_Check(o), name, " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

// Runs `body` with C++ exceptions turned into Python ones.
template <typename F>
PyObject* guarded(F&& body) {
    try {
        return body();
    } catch (python_error& e) {
        e.restore();
    } catch (const c10::ValueError& e) {
        PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* const torch_module = PyImport_ImportModule("torch");
        PyObject* const type = torch_module != nullptr ? PyObject_GetAttrString(torch_module, "OutOfMemoryError") : nullptr;
        PyErr_SetString(type != nullptr ? type : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch_module);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

}  // namespace penc_torch
