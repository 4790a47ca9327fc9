// The paged 4-bit cache's calls of tilemix_amd/_host.so (host_kv4.cpp).
#pragma once

#include <Python.h>

PyObject* kv4_bind(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_built_for(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_check(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_store(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_load(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_extend(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* kv4_truncate(PyObject*, PyObject* const* args, Py_ssize_t n);
