// Layer norm and products with an epilogue (native_operators.cpp), block-scaled products, norms around a residual add and the gradients' norm (native_blocks.cpp) as functions of the
// host extension.
#pragma once
#include <Python.h>

namespace native {

PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* add_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* epilogue(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* epilogue_prepared(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* block_scaled(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* gated_add_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* clip_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs);

}  // namespace native
