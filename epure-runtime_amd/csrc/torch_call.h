// What the native call paths share (torch_call.cpp, torch_paged.cpp,
// torch_draft.cpp).
#pragma once

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

#include <stdint.h>

#include "epure_hip.h"

namespace epure_torch {

extern decltype(&ep_last_error) fn_error;
extern PyObject *fn_stream;  // torch._C._cuda_getCurrentRawStream

// EP_F32 / EP_F16 / EP_BF16, or -1.
inline int dtype_code(at::ScalarType t)
{
    return t == at::kFloat ? EP_F32 : t == at::kHalf ? EP_F16 : t == at::kBFloat16 ? EP_BF16 : -1;
}
inline int dtype_code(const at::Tensor &t) { return dtype_code(t.scalar_type()); }

bool plain_call();
bool plain_tensor(PyObject *o);
void *stream_of(const at::Tensor &t, bool *ok);
at::Tensor bytes_like(const at::Tensor &t, size_t n);
PyObject *failed(const char *what, int rc);
bool args_are(Py_ssize_t n, Py_ssize_t want);

extern PyMethodDef paged_methods[];  // torch_paged.cpp
extern PyMethodDef draft_methods[];  // torch_draft.cpp

}  // namespace epure_torch
