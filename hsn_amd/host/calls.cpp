// The calls of a decoded token in one step from the interpreter: the language-model operators'
// Python mirrors (hsn_amd/scan.py, unit_layer.py, sampling.py) check their tensors, allocate outputs
// and workspace and call the C entry point through this module where it is built. Made in the
// interpreter, the checks, allocations and the conversion of some twenty arguments cost 4 to 6 us a
// call, more than the kernel of a single position; here they cost about 1 us.
//
// Every function takes the C entry points' addresses and the raw stream, and returns
//   None   a check failed: nothing was allocated or launched, and the caller makes the same checks in
//          Python, where each mismatch has its message;
//   int    the entry point's status, not HSN_OK;
//   else   the outputs.
// The tensors' device is current while an entry point runs: it launches on the current device, and the
// default stream's handle, 0, names no device.
// Host code only: nothing here runs on a device (CPython C API, linked against the installed PyTorch).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <initializer_list>

#include "../../include/hsn_sample.h"
#include "../../include/hsn_units_layer.h"

namespace {

using at::Tensor;
using P = const void*;

// One argument after the other.
struct Arguments {
    PyObject* const* at;
    PyObject* const* end;
    bool ok = true;

    PyObject* next() {
        if (at == end) {
            ok = false;
            return Py_None;
        }
        return *at++;
    }
    const Tensor* tensor() {  // null: None
        PyObject* o = next();
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) {
            ok = false;
            return nullptr;
        }
        return &THPVariable_Unpack(o);
    }
    int64_t integer() {
        PyObject* o = next();
        const int64_t v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
        if (!PyLong_Check(o) || (v == -1 && PyErr_Occurred())) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    double number() {
        const double v = PyFloat_AsDouble(next());
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
};

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}

// A tensor that the kernels can read at its address (no subclass with another storage).
bool plain(const Tensor& t) { return t.has_storage() && t.layout() == at::kStrided; }

// An absent tensor, or a contiguous one of this shape, type and device.
bool dense(const Tensor* t, at::IntArrayRef shape, at::ScalarType type, at::Device device) {
    return !t || (t->scalar_type() == type && t->device() == device && t->sizes() == shape && plain(*t) &&
                  t->is_contiguous());
}

// A tensor like `y` whose last dimension is contiguous.
bool like(const Tensor* t, const Tensor& y) {
    return t && t->scalar_type() == y.scalar_type() && t->device() == y.device() && t->sizes() == y.sizes() &&
           plain(*t) && (t->stride(-1) == 1 || t->size(-1) <= 1);
}

// Whether the caller wants a gradient with respect to one of these, for an operator that has none.
bool wants_gradient(std::initializer_list<const Tensor*> of) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : of)
        if (t && t->requires_grad()) return true;
    return false;
}

P address(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

template <typename F>
F entry(int64_t at) {
    return reinterpret_cast<F>(static_cast<uintptr_t>(at));
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

Tensor workspace(int64_t bytes, const at::TensorOptions& on) {
    return bytes ? at::empty({bytes}, on.dtype(at::kByte)) : Tensor();
}

// scan_forward(workspace, forward, stream, y, gate, reset, h0, candidate, save, span)
PyObject* scan_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *y = in.tensor(), *gate = in.tensor(), *reset = in.tensor(), *h0 = in.tensor();
    const int64_t candidate = in.integer(), save = in.integer(), span = in.integer();
    if (!in.ok || !y || y->dim() != 3 || !y->is_cuda() || y->size(2) < 1) Py_RETURN_NONE;
    const int code = dtype_code(y->scalar_type());
    const int64_t B = y->size(0), T = y->size(1), D = y->size(2);
    if (code < 0 || candidate < 0 || B > INT32_MAX || T > INT32_MAX || D > INT32_MAX || !like(y, *y) ||
        !like(gate, *y) || !dense(reset, {B, T}, at::kBool, y->device()) ||
        !dense(h0, {B, D}, at::kFloat, y->device()))
        Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int, int, int64_t*)>(size_at)(B, T, D, code, 0, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(y->device());
    const auto on = at::TensorOptions().device(y->device());
    const Tensor h = at::empty({B, T, D}, on.dtype(y->scalar_type()));
    const Tensor h_T = at::empty({B, D}, on.dtype(at::kFloat));
    Tensor marks;
    if (save) marks = at::empty({B, (T + span - 1) / span, D}, on.dtype(at::kFloat));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int64_t, P, int64_t, int64_t, int, int, P, P, P, P, P, int, int, int, P,
                           int64_t, P)>(call_at)(
        y->data_ptr(), y->stride(0), y->stride(1), gate->data_ptr(), gate->stride(0), gate->stride(1), code,
        candidate, address(reset), address(h0), h.data_ptr(), h_T.data_ptr(),
        save ? marks.data_ptr() : nullptr, B, T, D, bytes ? ws.data_ptr() : nullptr, bytes,
        entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return Py_BuildValue("(NNN)", wrap(h), wrap(h_T), wrap(marks));
    END_HANDLE_TH_ERRORS
}

// scan_backward(workspace, backward, stream, y, gate, marks, reset, d_h, d_h_T, candidate, span)
PyObject* scan_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *y = in.tensor(), *gate = in.tensor(), *marks = in.tensor(), *reset = in.tensor();
    const Tensor *d_h = in.tensor(), *d_h_T = in.tensor();
    const int64_t candidate = in.integer(), span = in.integer();
    if (!in.ok || !y || !marks || y->dim() != 3 || !y->is_cuda() || y->size(2) < 1) Py_RETURN_NONE;
    const int code = dtype_code(y->scalar_type());
    const int64_t B = y->size(0), T = y->size(1), D = y->size(2);
    if (code < 0 || candidate < 0 || B > INT32_MAX || T > INT32_MAX || D > INT32_MAX || !like(y, *y) ||
        !like(gate, *y) || (d_h && !like(d_h, *y)) ||
        !dense(marks, {B, (T + span - 1) / span, D}, at::kFloat, y->device()) ||
        !dense(reset, {B, T}, at::kBool, y->device()) || !dense(d_h_T, {B, D}, at::kFloat, y->device()))
        Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int, int, int64_t*)>(size_at)(B, T, D, code, 1, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(y->device());
    const auto on = at::TensorOptions().device(y->device());
    const Tensor d_y = at::empty({B, T, D}, on.dtype(y->scalar_type()));
    const Tensor d_gate = at::empty({B, T, D}, on.dtype(y->scalar_type()));
    const Tensor d_h0 = at::empty({B, D}, on.dtype(at::kFloat));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int64_t, P, int64_t, int64_t, int, int, P, P, P, int64_t, int64_t, P, P,
                           P, P, int, int, int, P, int64_t, P)>(call_at)(
        y->data_ptr(), y->stride(0), y->stride(1), gate->data_ptr(), gate->stride(0), gate->stride(1), code,
        candidate, address(reset), marks->data_ptr(), address(d_h), d_h ? d_h->stride(0) : 0,
        d_h ? d_h->stride(1) : 0, address(d_h_T), d_y.data_ptr(), d_gate.data_ptr(), d_h0.data_ptr(), B, T, D,
        bytes ? ws.data_ptr() : nullptr, bytes, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return Py_BuildValue("(NNN)", wrap(d_y), wrap(d_gate), wrap(d_h0));
    END_HANDLE_TH_ERRORS
}

// scan_step(step, stream, y, gate, state, rows, reset, candidate)
PyObject* scan_step(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t call_at = in.integer(), stream = in.integer();
    const Tensor *y = in.tensor(), *gate = in.tensor(), *state = in.tensor(), *rows = in.tensor();
    const Tensor* reset = in.tensor();
    const int64_t candidate = in.integer();
    if (!in.ok || !y || !state || y->dim() != 2 || state->dim() != 2 || !y->is_cuda() || y->size(1) < 1)
        Py_RETURN_NONE;
    const int code = dtype_code(y->scalar_type());
    const int64_t n = y->size(0), D = y->size(1), S = state->size(0);
    if (code < 0 || candidate < 0 || n > INT32_MAX || D > INT32_MAX || S > INT32_MAX || !like(y, *y) ||
        !like(gate, *y) || !dense(state, {S, D}, at::kFloat, y->device()) ||
        !dense(rows, {n}, at::kInt, y->device()) || !dense(reset, {n}, at::kBool, y->device()) ||
        wants_gradient({y, gate, state}))
        Py_RETURN_NONE;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(y->device());
    const Tensor h = at::empty({n, D}, at::TensorOptions().device(y->device()).dtype(y->scalar_type()));
    const int status = entry<int (*)(P, int64_t, P, int64_t, int, int, P, P, P, P, int, int, int, P)>(call_at)(
        y->data_ptr(), y->stride(0), gate->data_ptr(), gate->stride(0), code, candidate, address(rows),
        address(reset), state->data_ptr(), h.data_ptr(), n, S, D, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    // an update in place, as autograd sees it; an inference tensor has no version
    if (n && !state->is_inference()) state->unsafeGetTensorImpl()->bump_version();
    return wrap(h);
    END_HANDLE_TH_ERRORS
}

// unit_layer(workspace, layer, stream, x, router, W1, b1, W2, b2, k, activation, gated)
PyObject* unit_layer(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *x = in.tensor(), *router = in.tensor(), *W1 = in.tensor(), *b1 = in.tensor();
    const Tensor *W2 = in.tensor(), *b2 = in.tensor();
    const int64_t k = in.integer(), activation = in.integer(), gated = in.integer();
    if (!in.ok || !x || !router || !W1 || !W2 || x->dim() != 2 || W2->dim() != 3 || !x->is_cuda() ||
        activation < 0)
        Py_RETURN_NONE;
    const auto type = x->scalar_type();
    const auto device = x->device();
    const int code = dtype_code(type);
    const int64_t n = x->size(0), d_in = x->size(1), M = W2->size(0), H = W2->size(1), d_out = W2->size(2);
    const int64_t H1 = gated ? 2 * H : H;
    if (code < 0 || !like(x, *x) || k < 1 || k > M || k > HSN_UNITS_MAX_CHOSEN ||
        n > HSN_UNITS_MAX_TOKENS || M > HSN_UNITS_MAX || d_in > 65536 || H > 65536 ||
        d_out > 65536 || !dense(router, {M, d_in}, type, device) || !dense(W1, {M, d_in, H1}, type, device) ||
        !dense(b1, {M, H1}, type, device) || !dense(W2, {M, H, d_out}, type, device) ||
        !dense(b2, {M, d_out}, type, device))
        Py_RETURN_NONE;
    if (wants_gradient({x, router, W1, b1, W2, b2})) Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int, int, int, int, int, int64_t*)>(size_at)(
        n, M, k, d_in, H, d_out, code, activation, &bytes);
    if (status) return PyLong_FromLong(status);
    const c10::DeviceGuard current(device);
    const auto on = at::TensorOptions().device(device);
    const Tensor y = at::empty({n, d_out}, on.dtype(type));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, P, P, P, P, P, P, int, int, int, int, int, int, int, int, P, int64_t,
                           P)>(call_at)(
        x->data_ptr(), x->stride(0), router->data_ptr(), W1->data_ptr(), address(b1), W2->data_ptr(),
        address(b2), y.data_ptr(), n, M, k, d_in, H, d_out, code, activation, bytes ? ws.data_ptr() : nullptr,
        bytes, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(y);
    END_HANDLE_TH_ERRORS
}

struct Settings {  // hsn_sample_settings
    float temperature;
    int32_t top_k;
    float top_p, min_p;
};

// sample(workspace, sample, stream, logits, u, temperature, top_k, top_p, min_p)
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *logits = in.tensor(), *u = in.tensor();
    if (!in.ok || !logits || !u || logits->dim() != 2 || !logits->is_cuda()) Py_RETURN_NONE;
    const int code = dtype_code(logits->scalar_type());
    const auto device = logits->device();
    const int64_t n = logits->size(0), V = logits->size(1);
    if (code < 0 || n > INT32_MAX || V < 1 || V > HSN_SAMPLE_MAX_TOKENS || !like(logits, *logits) ||
        !dense(u, {n}, at::kFloat, device))
        Py_RETURN_NONE;
    // a setting: a row's values in a tensor, or one number
    const Tensor* rows[4] = {};
    Settings settings{};
    for (int i = 0; i < 4; ++i) {
        const bool whole = i == 1;
        if (in.at != in.end && THPVariable_Check(*in.at)) {
            rows[i] = in.tensor();
            if (!dense(rows[i], {n}, whole ? at::kInt : at::kFloat, device)) Py_RETURN_NONE;
        } else if (whole) {
            const int64_t k = in.integer();
            if (!in.ok || k < 0 || k > INT32_MAX) Py_RETURN_NONE;
            settings.top_k = static_cast<int32_t>(k);
        } else {
            const float v = static_cast<float>(in.number());
            (i == 0 ? settings.temperature : i == 2 ? settings.top_p : settings.min_p) = v;
        }
    }
    if (!in.ok) Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int64_t*)>(size_at)(n, V, code, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(device);
    const auto on = at::TensorOptions().device(device);
    const Tensor tokens = at::empty({n}, on.dtype(at::kLong));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int, P, P, P, P, P, P, P, int, int, P, int64_t, P)>(call_at)(
        logits->data_ptr(), logits->stride(0), code, u->data_ptr(), address(rows[0]), address(rows[1]),
        address(rows[2]), address(rows[3]), &settings, tokens.data_ptr(), n, V,
        bytes ? ws.data_ptr() : nullptr, bytes, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(tokens);
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef kMethods[] = {
    {"scan_forward", fast<scan_forward>(), METH_FASTCALL,
     "(workspace, forward, stream, y, gate, reset, h0, candidate, save, span) -> (h, h_T, marks)"},
    {"scan_backward", fast<scan_backward>(), METH_FASTCALL,
     "(workspace, backward, stream, y, gate, marks, reset, d_h, d_h_T, candidate, span) -> (d_y, d_gate, "
     "d_h0)"},
    {"scan_step", fast<scan_step>(), METH_FASTCALL,
     "(step, stream, y, gate, state, rows, reset, candidate) -> h"},
    {"unit_layer", fast<unit_layer>(), METH_FASTCALL,
     "(workspace, layer, stream, x, router, W1, b1, W2, b2, k, activation, gated) -> y"},
    {"sample", fast<sample>(), METH_FASTCALL,
     "(workspace, sample, stream, logits, u, temperature, top_k, top_p, min_p) -> tokens"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_calls",
                       "The language-model operators' calls in one step (host code only).", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&kModule); }
