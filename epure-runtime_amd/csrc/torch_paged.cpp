// Python calls of the paged-cache operators (include/epure_paged.h) on plain
// GPU tensors, one native call each, as torch_call.cpp does for the packed
// linears: through ctypes a token's rotation spent 17 us around a 3 us kernel.
// What is out of the ordinary (another type, layout or device, a torch mode,
// an empty call, an argument to refuse) returns NotImplemented, and the caller
// takes the way through Python (epure/paged.py), which checks and raises.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>

#include "torch_call.h"
#include "epure_paged.h"

namespace epure_torch {
namespace {

decltype(&ep_rotate) fn_rotate;
decltype(&ep_kv_append) fn_append;
decltype(&ep_kv_read) fn_read;
decltype(&ep_paged_attention_workspace) fn_attend_ws;
decltype(&ep_paged_attention) fn_attend;

// A plain GPU tensor argument on `dev` (any where dev < 0), or nullptr.  One
// with a forward-mode tangent is not plain: nothing here would carry it on.
const at::Tensor *gpu_tensor(PyObject *o, c10::DeviceIndex &dev)
{
    if (!plain_tensor(o))
        return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || (dev >= 0 && t.get_device() != dev) || t._fw_grad(0).defined())
        return nullptr;
    dev = t.get_device();
    return &t;
}

// [B, S, heads, D] of a served type, each head's values adjacent, none empty.
bool heads_ok(const at::Tensor &t)
{
    return t.dim() == 4 && t.numel() > 0 && dtype_code(t) >= 0 && (t.stride(3) == 1 || t.size(3) == 1);
}

ep_heads heads_of(const at::Tensor &t)
{
    return ep_heads{t.data_ptr(), dtype_code(t), (int)t.size(2), t.stride(0), t.stride(1), t.stride(2)};
}

// positions broadcast to [B, S]; false where they are not int64 or do not.
bool tokens_of(const at::Tensor &pos, int64_t B, int64_t S, ep_tokens &t)
{
    const int64_t d = pos.dim();
    if (pos.scalar_type() != at::kLong || d > 2)
        return false;
    const int64_t want[2] = {B, S};
    int64_t stride[2] = {0, 0};
    for (int64_t i = 0; i < d; ++i) {
        const int64_t at = 2 - d + i;
        if (pos.size(i) != want[at] && pos.size(i) != 1)
            return false;
        stride[at] = pos.size(i) == 1 ? 0 : pos.stride(i);
    }
    t = ep_tokens{B, S, (const int64_t *)pos.const_data_ptr(), stride[0], stride[1], nullptr, 0, 0};
    return true;
}

bool table_of(const at::Tensor &table, ep_tokens &t)
{
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != t.B ||
        (table.size(1) > 1 && table.stride(1) != 1))
        return false;
    t.table = (const int32_t *)table.const_data_ptr();
    t.table_stride = table.stride(0);
    t.width = table.size(1);
    return true;
}

bool needs_grad(std::initializer_list<const at::Tensor *> ts)
{
    if (!c10::GradMode::is_enabled())
        return false;
    for (const at::Tensor *t : ts)
        if (t && t->requires_grad())
            return true;
    return false;
}

// The cache of arguments k, v, k_scale, v_scale (None in a 16-bit one).
bool cache_of(PyObject *const *args, c10::DeviceIndex &dev, ep_kv_cache &c)
{
    const at::Tensor *k = gpu_tensor(args[0], dev), *v = k ? gpu_tensor(args[1], dev) : nullptr;
    if (!v || k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() ||
        !k->is_contiguous() || !v->is_contiguous() || needs_grad({k, v}))
        return false;
    const auto dt = k->scalar_type();
    const int code = dt == at::kChar ? EP_I8 : dt == at::kFloat8_e4m3fn ? EP_E4M3 : dtype_code(dt);
    if (code < 0 || code == EP_F32)
        return false;
    float *scale[2] = {nullptr, nullptr};
    if (code == EP_I8 || code == EP_E4M3)
        for (int i = 0; i < 2; ++i) {
            const at::Tensor *s = gpu_tensor(args[2 + i], dev);
            if (!s || s->scalar_type() != at::kFloat || !s->is_contiguous() || s->sizes() != k->sizes().slice(0, 3) ||
                needs_grad({s}))
                return false;
            scale[i] = (float *)s->data_ptr();
        }
    c = ep_kv_cache{k->data_ptr(), v->data_ptr(), scale[0], scale[1], code,
                    (int)k->size(1), (int)k->size(2), (int)k->size(3), k->size(0)};
    return true;
}

bool rotation_of(const at::Tensor *cos, const at::Tensor *sin, bool interleaved, ep_rotation &r)
{
    if (!cos || !sin || cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || cos->dim() != 2 ||
        sin->sizes() != cos->sizes() || !cos->is_contiguous() || !sin->is_contiguous())
        return false;
    r = ep_rotation{(const float *)cos->const_data_ptr(), (const float *)sin->const_data_ptr(), cos->size(0),
                    (int)(2 * cos->size(1)), interleaved};
    return true;
}

at::Tensor like(const at::Tensor &t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

// ------------------------------------------------------------------ rotation
// What a rotation's gradient needs of it.  The engine runs a node's backward
// pass on the stream of its forward pass (from a thread that does not hold the
// interpreter's lock), so that stream is kept rather than asked for.
struct Turn {
    at::Tensor positions, cos, sin;
    bool interleaved, inverse;
    void *stream;

    void save(torch::autograd::AutogradContext *ctx) const
    {
        ctx->save_for_backward({positions, cos, sin});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["stream"] = (int64_t)stream;
    }
    // The way back of a saved turn.
    static Turn back(torch::autograd::AutogradContext *ctx)
    {
        const auto s = ctx->get_saved_variables();
        return Turn{s[0], s[1], s[2], ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool(),
                    (void *)ctx->saved_data["stream"].toInt()};
    }
};

// q and k (undefined: none) turned.
int turn(const at::Tensor &q, const at::Tensor &k, const Turn &t, at::Tensor &qo, at::Tensor &ko)
{
    ep_rotation r;
    ep_tokens tok;
    TORCH_CHECK(rotation_of(&t.cos, &t.sin, t.interleaved, r) && tokens_of(t.positions, q.size(0), q.size(1), tok),
                "rotation: tables or positions changed");
    const at::Tensor qs = q.stride(3) == 1 || q.size(3) == 1 ? q : q.contiguous();
    const at::Tensor ks = !k.defined() || k.stride(3) == 1 || k.size(3) == 1 ? k : k.contiguous();
    qo = like(q);
    if (k.defined())
        ko = like(k);
    const ep_heads qh = heads_of(qs), kh = k.defined() ? heads_of(ks) : ep_heads{};
    return fn_rotate(&qh, k.defined() ? &kh : nullptr, &r, &tok, q.size(3), t.inverse, qo.data_ptr(),
                     k.defined() ? ko.data_ptr() : nullptr, t.stream);
}

void turned(int rc)
{
    TORCH_CHECK_VALUE(rc <= 0, "ep_rotate declined: ", fn_error());
    TORCH_CHECK(rc == EP_OK, "ep_rotate failed (", rc, "): ", fn_error());
}

// One tensor, or two of a call, turned; the gradient of a turn is the turn
// the other way, and differentiable likewise.
struct RotateOne : torch::autograd::Function<RotateOne> {
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const Turn &t)
    {
        t.save(ctx);
        at::Tensor y, none;
        turned(turn(x, none, t, y, none));
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                   torch::autograd::variable_list g)
    {
        return {RotateOne::apply(g[0], Turn::back(ctx)), at::Tensor()};
    }
};

// Two: the output of an input that needs no gradient is a constant.
struct RotateTwo : torch::autograd::Function<RotateTwo> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &q,
                                                  const at::Tensor &k, const Turn &t)
    {
        ctx->set_materialize_grads(false);
        t.save(ctx);
        at::Tensor qo, ko;
        turned(turn(q, k, t, qo, ko));
        if (!q.requires_grad())
            ctx->mark_non_differentiable({qo});
        if (!k.requires_grad())
            ctx->mark_non_differentiable({ko});
        return {qo, ko};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                   torch::autograd::variable_list g)
    {
        const Turn t = Turn::back(ctx);
        torch::autograd::variable_list r(3);
        if (g[0].defined() && g[1].defined()) {
            const auto two = RotateTwo::apply(g[0], g[1], t);
            r[0] = two[0];
            r[1] = two[1];
        } else
            for (int i = 0; i < 2; ++i)
                if (g[i].defined())
                    r[i] = RotateOne::apply(g[i], t);
        return r;
    }
};

// rotate(q, k or None, positions, cos, sin, interleaved): (q', k') or, without
// k, q'.
PyObject *rotate(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (!args_are(nargs, 6))
        return nullptr;
    if (!plain_call())
        Py_RETURN_NOTIMPLEMENTED;
    c10::DeviceIndex dev = -1;
    const bool two = args[1] != Py_None;
    const at::Tensor *q = gpu_tensor(args[0], dev), *k = two && q ? gpu_tensor(args[1], dev) : nullptr;
    const at::Tensor *pos = q ? gpu_tensor(args[2], dev) : nullptr, *cos = q ? gpu_tensor(args[3], dev) : nullptr;
    const at::Tensor *sin = q ? gpu_tensor(args[4], dev) : nullptr;
    const int interleaved = PyObject_IsTrue(args[5]);
    if (interleaved < 0)
        return nullptr;
    ep_rotation r;
    ep_tokens tok;
    if (!q || !pos || !heads_ok(*q) || !tokens_of(*pos, q->size(0), q->size(1), tok) ||
        !rotation_of(cos, sin, interleaved, r) || r.dim > q->size(3))
        Py_RETURN_NOTIMPLEMENTED;
    if (two && (!k || !heads_ok(*k) || k->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) ||
                k->size(1) != q->size(1) || k->size(3) != q->size(3)))
        Py_RETURN_NOTIMPLEMENTED;
    bool ok;
    void *stream = stream_of(*q, &ok);
    if (!ok)
        return nullptr;
    const Turn t{*pos, *cos, *sin, (bool)interleaved, false, stream};
    at::Tensor qo, ko;
    if (!needs_grad({q, k})) {
        const int rc = turn(*q, two ? *k : at::Tensor(), t, qo, ko);
        if (rc > 0)
            Py_RETURN_NOTIMPLEMENTED;
        if (rc < 0)
            return failed("ep_rotate", rc);
    } else if (two) {
        const auto y = RotateTwo::apply(*q, *k, t);
        qo = y[0];
        ko = y[1];
    } else
        qo = RotateOne::apply(*q, t);
    PyObject *a = THPVariable_Wrap(qo);
    if (!two || !a)
        return a;
    PyObject *b = THPVariable_Wrap(ko), *pair = b ? PyTuple_New(2) : nullptr;
    if (!pair) {
        Py_DECREF(a);
        Py_XDECREF(b);
        return nullptr;
    }
    PyTuple_SET_ITEM(pair, 0, a);
    PyTuple_SET_ITEM(pair, 1, b);
    return pair;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ the cache
// append(k, v, positions, table, q or None, cos or None, sin or None,
// interleaved, cache k, v, k_scale, v_scale): q turned, or None.
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (!args_are(nargs, 12))
        return nullptr;
    if (!plain_call())
        Py_RETURN_NOTIMPLEMENTED;
    c10::DeviceIndex dev = -1;
    ep_kv_cache c;
    if (!cache_of(args + 8, dev, c))
        Py_RETURN_NOTIMPLEMENTED;
    const bool some_q = args[4] != Py_None, turns = args[5] != Py_None;
    const at::Tensor *k = gpu_tensor(args[0], dev), *v = gpu_tensor(args[1], dev), *pos = gpu_tensor(args[2], dev);
    const at::Tensor *table = gpu_tensor(args[3], dev), *q = some_q ? gpu_tensor(args[4], dev) : nullptr;
    const int interleaved = PyObject_IsTrue(args[7]);
    if (interleaved < 0)
        return nullptr;
    ep_tokens tok;
    ep_rotation r;
    if (!k || !v || !pos || !table || !heads_ok(*k) || !heads_ok(*v) || k->sizes() != v->sizes() ||
        k->scalar_type() != v->scalar_type() || k->size(2) != c.heads || k->size(3) != c.D ||
        !tokens_of(*pos, k->size(0), k->size(1), tok) || !table_of(*table, tok) || needs_grad({q, k, v}))
        Py_RETURN_NOTIMPLEMENTED;
    if (some_q && (!q || !heads_ok(*q) || q->scalar_type() != k->scalar_type() || q->size(0) != k->size(0) ||
                   q->size(1) != k->size(1) || q->size(3) != c.D))
        Py_RETURN_NOTIMPLEMENTED;
    if (turns && (!rotation_of(gpu_tensor(args[5], dev), gpu_tensor(args[6], dev), interleaved, r) || r.dim > c.D))
        Py_RETURN_NOTIMPLEMENTED;
    bool ok;
    void *stream = stream_of(*k, &ok);
    if (!ok)
        return nullptr;
    const at::Tensor qo = some_q ? like(*q) : at::Tensor();
    const ep_heads qh = some_q ? heads_of(*q) : ep_heads{}, kh = heads_of(*k), vh = heads_of(*v);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn_append(some_q ? &qh : nullptr, &kh, &vh, turns ? &r : nullptr, &tok, &c, some_q ? qo.data_ptr() : nullptr,
                   stream);
    Py_END_ALLOW_THREADS
    if (rc > 0)
        Py_RETURN_NOTIMPLEMENTED;
    if (rc < 0)
        return failed("ep_kv_append", rc);
    if (!some_q)
        Py_RETURN_NONE;
    return THPVariable_Wrap(qo);
    END_HANDLE_TH_ERRORS
}

// read(positions, table, dtype, cache k, v, k_scale, v_scale): (k, v)
PyObject *read(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (!args_are(nargs, 7))
        return nullptr;
    if (!plain_call() || !THPDtype_Check(args[2]))
        Py_RETURN_NOTIMPLEMENTED;
    c10::DeviceIndex dev = -1;
    ep_kv_cache c;
    if (!cache_of(args + 3, dev, c))
        Py_RETURN_NOTIMPLEMENTED;
    const at::Tensor *pos = gpu_tensor(args[0], dev), *table = gpu_tensor(args[1], dev);
    const auto dtype = ((THPDtype *)args[2])->scalar_type;
    ep_tokens tok;
    if (!pos || !table || pos->dim() != 2 || pos->numel() == 0 || dtype_code(dtype) < 0 ||
        !tokens_of(*pos, pos->size(0), pos->size(1), tok) || !table_of(*table, tok))
        Py_RETURN_NOTIMPLEMENTED;
    bool ok;
    void *stream = stream_of(*pos, &ok);
    if (!ok)
        return nullptr;
    at::Tensor out[2];
    for (at::Tensor &t : out)
        t = at::empty({tok.B, tok.S, c.heads, c.D}, pos->options().dtype(dtype));
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn_read(&tok, &c, out[0].data_ptr(), out[1].data_ptr(), dtype_code(dtype), stream);
    Py_END_ALLOW_THREADS
    if (rc > 0)
        Py_RETURN_NOTIMPLEMENTED;
    if (rc < 0)
        return failed("ep_kv_read", rc);
    PyObject *a = THPVariable_Wrap(out[0]), *b = a ? THPVariable_Wrap(out[1]) : nullptr, *t = b ? PyTuple_New(2) : nullptr;
    if (!t) {
        Py_XDECREF(a);
        Py_XDECREF(b);
        return nullptr;
    }
    PyTuple_SET_ITEM(t, 0, a);
    PyTuple_SET_ITEM(t, 1, b);
    return t;
    END_HANDLE_TH_ERRORS
}

// attend(q, positions, table, scale or None, window or None, cache k, v,
// k_scale, v_scale): the attention's output
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (!args_are(nargs, 9))
        return nullptr;
    if (!plain_call())
        Py_RETURN_NOTIMPLEMENTED;
    c10::DeviceIndex dev = -1;
    ep_kv_cache c;
    if (!cache_of(args + 5, dev, c))
        Py_RETURN_NOTIMPLEMENTED;
    const at::Tensor *q = gpu_tensor(args[0], dev), *pos = gpu_tensor(args[1], dev), *table = gpu_tensor(args[2], dev);
    ep_tokens tok;
    if (!q || !pos || !table || !heads_ok(*q) || q->size(3) != c.D ||
        !tokens_of(*pos, q->size(0), q->size(1), tok) || !table_of(*table, tok) || needs_grad({q}))
        Py_RETURN_NOTIMPLEMENTED;
    const double scale = args[3] == Py_None ? 1.0 / std::sqrt((double)c.D) : PyFloat_AsDouble(args[3]);
    const int64_t window = args[4] == Py_None ? 0 : PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NOTIMPLEMENTED;
    }
    if (args[4] != Py_None && window < 1)
        Py_RETURN_NOTIMPLEMENTED;
    bool ok;
    void *stream = stream_of(*q, &ok);
    if (!ok)
        return nullptr;
    const ep_heads qh = heads_of(*q);
    const size_t n = fn_attend_ws(&qh, &tok, &c);
    const at::Tensor out = like(*q), ws = bytes_like(*q, n);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn_attend(&qh, &tok, &c, (float)scale, window, out.data_ptr(), n ? ws.data_ptr() : nullptr, n, stream);
    Py_END_ALLOW_THREADS
    if (rc == EP_ERR_ARG || rc > 0)     // heads that do not divide, q's type or alignment
        Py_RETURN_NOTIMPLEMENTED;
    if (rc < 0)
        return failed("ep_paged_attention", rc);
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// bind_paged(rotate, append, read, attention_workspace, attention): addresses
PyObject *bind_paged(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    if (!args_are(nargs, 5))
        return nullptr;
    fn_rotate = (decltype(fn_rotate))PyLong_AsVoidPtr(args[0]);
    fn_append = (decltype(fn_append))PyLong_AsVoidPtr(args[1]);
    fn_read = (decltype(fn_read))PyLong_AsVoidPtr(args[2]);
    fn_attend_ws = (decltype(fn_attend_ws))PyLong_AsVoidPtr(args[3]);
    fn_attend = (decltype(fn_attend))PyLong_AsVoidPtr(args[4]);
    if (PyErr_Occurred())
        return nullptr;
    Py_RETURN_NONE;
}

}  // namespace

PyMethodDef paged_methods[] = {
    {"bind_paged", (PyCFunction)(void (*)(void))bind_paged, METH_FASTCALL, nullptr},
    {"rotate", (PyCFunction)(void (*)(void))rotate, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"read", (PyCFunction)(void (*)(void))read, METH_FASTCALL, nullptr},
    {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace epure_torch
