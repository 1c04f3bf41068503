// What the methods that go from Python's tensors to the library have in common (host code).
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstdint>
#include <optional>

#include "../../include/fmoe_hip.h"

namespace fmoe_call {

inline int dtype_code(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FMOE_F32;
        case at::kBFloat16: return FMOE_BF16;
        case at::kHalf: return FMOE_F16;
        default: return -1;
    }
}
inline void *pointer(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline at::Tensor same(const at::Tensor &t) { return at::empty(t.sizes(), t.options()); }

using Maybe = std::optional<at::Tensor>;   // (what a node takes where there may be no tensor)
inline Maybe maybe(const at::Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }

// The interpreter's lock, given back while this lives: an allocation may wait for the device, a launch for a full queue
struct WithoutLock {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutLock() { PyEval_RestoreThread(state); }
};

// The first N arguments as tensors (undefined for None); false, with an exception set, where one is neither
template <size_t N> bool tensors(PyObject *const *args, std::array<at::Tensor, N> &t) {
    for (size_t i = 0; i < N; ++i) {
        if (args[i] == Py_None) continue;
        if (!THPVariable_Check(args[i])) {
            PyErr_SetString(PyExc_TypeError, "tensors or None");
            return false;
        }
        t[i] = THPVariable_Unpack(args[i]);
    }
    return true;
}
// The number behind them; false, with an exception set, where it is none
inline bool number(PyObject *arg, long &n) {
    n = PyLong_AsLong(arg);
    return n != -1 || !PyErr_Occurred();
}
// (a tensor without memory of its own, as some wrappers are, has a null pointer, which a parameter that is left out has too)
inline bool on_gpu(const at::Tensor &t) {
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg() && t.has_storage() &&
           (t.numel() == 0 || t.storage().data() != nullptr);
}

inline PyObject *wrap_or_none(at::Tensor t) {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
}

}  // namespace fmoe_call
