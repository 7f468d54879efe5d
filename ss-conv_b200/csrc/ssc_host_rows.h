// Python entry points of ssc_host_rows.cpp.
#pragma once
#include <Python.h>

PyObject *ssc_py_group_norm(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *ssc_py_gated_ff(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *ssc_py_row_operators(PyObject *, PyObject *const *args, Py_ssize_t n);
