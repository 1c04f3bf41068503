// Methods that block_call.cpp and expert_call.cpp add to the extension module of layer_call.cpp (host code).
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

PyObject *fmoe_block_bind(PyObject *, PyObject *args);
PyObject *fmoe_block_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *fmoe_block_balance_loss(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *fmoe_block_checkpoint_forward(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *fmoe_block_checkpoint_backward(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *fmoe_expert_bind(PyObject *, PyObject *args);
PyObject *fmoe_expert_gated_mlp(PyObject *, PyObject *const *args, Py_ssize_t n_args);
PyObject *fmoe_expert_linear_int8(PyObject *, PyObject *const *args, Py_ssize_t n_args);
