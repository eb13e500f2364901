// The verification of drafted tokens (include/epure_draft.h) on plain GPU
// tensors, one native call, as torch_paged.cpp does for the paged cache: what is
// out of the ordinary returns NotImplemented, and the caller takes the way
// through Python (epure/drafts.py), which checks and raises.
#include <c10/core/DeviceGuard.h>

#include "torch_call.h"
#include "epure_draft.h"

namespace epure_torch {
namespace {

decltype(&ep_verify_draft_workspace) fn_verify_ws;
decltype(&ep_verify_draft) fn_verify;

const at::Tensor *gpu(PyObject *o, int64_t dims, c10::DeviceIndex &dev)
{
    if (!plain_tensor(o))
        return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || (dev >= 0 && t.get_device() != dev) || t.dim() != dims)
        return nullptr;
    dev = t.get_device();
    return &t;
}

bool adjacent(const at::Tensor &t) { return t.stride(2) == 1 || t.size(2) == 1; }

// verify(target, drafted, uniforms, draft or None): (accepted, tokens)
PyObject *verify(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (!args_are(nargs, 4))
        return nullptr;
    if (!plain_call())
        Py_RETURN_NOTIMPLEMENTED;
    c10::DeviceIndex dev = -1;
    const bool given = args[3] != Py_None;
    const at::Tensor *target = gpu(args[0], 3, dev), *drafted = gpu(args[1], 2, dev), *u = gpu(args[2], 2, dev);
    const at::Tensor *draft = given ? gpu(args[3], 3, dev) : nullptr;
    if (!target || !drafted || !u || (given && !draft))
        Py_RETURN_NOTIMPLEMENTED;
    const int64_t B = target->size(0), n = drafted->size(1), V = target->size(2);
    if (dtype_code(*target) < 0 || drafted->scalar_type() != at::kLong || u->scalar_type() != at::kFloat || B < 1 ||
        n < 1 || n > 0x3fffffff || V < 1 || target->size(1) != n + 1 || drafted->size(0) != B || u->size(0) != B ||
        u->size(1) != n + 1 || !adjacent(*target))
        Py_RETURN_NOTIMPLEMENTED;
    if (given && (draft->scalar_type() != target->scalar_type() || draft->size(0) != B || draft->size(1) != n ||
                  draft->size(2) != V || !adjacent(*draft)))
        Py_RETURN_NOTIMPLEMENTED;
    bool ok;
    void *stream = stream_of(*target, &ok);
    if (!ok)
        return nullptr;
    const c10::DeviceGuard guard(target->device());
    const ep_draft d{B, V, (int)n, dtype_code(*target), target->const_data_ptr(), target->stride(0), target->stride(1),
                     given ? draft->const_data_ptr() : nullptr, given ? draft->stride(0) : 0, given ? draft->stride(1) : 0,
                     (const int64_t *)drafted->const_data_ptr(), drafted->stride(0), drafted->stride(1),
                     (const float *)u->const_data_ptr(), u->stride(0), u->stride(1)};
    const size_t bytes = fn_verify_ws(&d);
    const auto whole = drafted->options().requires_grad(false);
    const at::Tensor accepted = at::empty({B}, whole), tokens = at::empty({B, n + 1}, whole), ws = bytes_like(*drafted, bytes);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn_verify(&d, (int64_t *)accepted.data_ptr(), (int64_t *)tokens.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                   stream);
    Py_END_ALLOW_THREADS
    if (rc == EP_ERR_ARG || rc > 0)
        Py_RETURN_NOTIMPLEMENTED;
    if (rc < 0)
        return failed("ep_verify_draft", rc);
    PyObject *a = THPVariable_Wrap(accepted), *b = a ? THPVariable_Wrap(tokens) : nullptr, *pair = b ? PyTuple_New(2) : nullptr;
    if (!pair) {
        Py_XDECREF(a);
        Py_XDECREF(b);
        return nullptr;
    }
    PyTuple_SET_ITEM(pair, 0, a);
    PyTuple_SET_ITEM(pair, 1, b);
    return pair;
    END_HANDLE_TH_ERRORS
}

// bind_draft(workspace, verification): addresses
PyObject *bind_draft(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    if (!args_are(nargs, 2))
        return nullptr;
    fn_verify_ws = (decltype(fn_verify_ws))PyLong_AsVoidPtr(args[0]);
    fn_verify = (decltype(fn_verify))PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred())
        return nullptr;
    Py_RETURN_NONE;
}

}  // namespace

PyMethodDef draft_methods[] = {
    {"bind_draft", (PyCFunction)(void (*)(void))bind_draft, METH_FASTCALL, nullptr},
    {"verify", (PyCFunction)(void (*)(void))verify, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace epure_torch
