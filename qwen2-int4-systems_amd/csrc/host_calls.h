// Functions of the CPython module qwen_int4_hip._host, one source each group.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

PyObject* host_paged_append(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* host_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* host_verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t count);
