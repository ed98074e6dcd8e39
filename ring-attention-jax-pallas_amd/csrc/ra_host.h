// What the sources of the host extension share.
#pragma once
#include <Python.h>
#include <ATen/ATen.h>

namespace ra_host {

void check(const char* what, int code);       // raises what a library call's code says
void* stream(const at::Device& device);       // the current one
int row_dtype(at::ScalarType t);              // RA_DTYPE_*, -1 for others
const at::Tensor& tensor_of(PyObject* x);
PyObject* tuple_of(std::vector<at::Tensor>&& tensors);
PyMethodDef* paged_methods();

}  // namespace ra_host
