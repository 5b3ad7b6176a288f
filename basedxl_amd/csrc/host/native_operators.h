// Layer norm and products with an epilogue as functions of the host extension (native_operators.cpp).
#pragma once
#include <Python.h>

namespace native {

PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* add_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* epilogue(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* epilogue_prepared(PyObject*, PyObject* const* args, Py_ssize_t nargs);

}  // namespace native
