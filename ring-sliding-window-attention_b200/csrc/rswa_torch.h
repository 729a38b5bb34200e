// What the translation units of _native.so share.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>

#include <cstdint>

namespace rswa_host {

// The device's status word, or null where none has been made yet (new_status).
int32_t* status_word(int device);
// Whether a kernel of an earlier call has reported an error that nobody has been told of yet.
bool reported(int device);
// Raises what a return code of the C ABI stands for.
void check(int rc, const char* what);

PyObject* py_cache_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_cache_read(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_cache_attn(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_weight_sums(PyObject*, PyObject* const* args, Py_ssize_t n);

}  // namespace rswa_host
