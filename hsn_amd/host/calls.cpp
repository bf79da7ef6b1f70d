// The calls of a decoded token and of a training step's operators in one step from the interpreter: the
// language-model operators' Python mirrors (hsn_amd/scan.py, unit_layer.py, sampling.py, embedding.py,
// scoring.py, unit_router.py, grad_clip.py) check their tensors, allocate outputs and workspace and call
// the C entry point through this module where it is built. Made in the interpreter, the checks,
// allocations and the conversion of some twenty arguments cost 4 to 6 us a call, more than the kernel of a
// single position; here they cost about 1 us.
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
#include <vector>

#include "../../include/hsn_embed.h"
#include "../../include/hsn_sample.h"
#include "../../include/hsn_score.h"
#include "../../include/hsn_unit_router.h"
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

// A tensor that the kernels can read at its address (no subclass with another storage, no negated view).
bool plain(const Tensor& t) { return t.has_storage() && t.layout() == at::kStrided && !t.is_neg(); }

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

// Tokens of any shape as B rows of T; a shape that is neither is not `ok`.
struct Tokens {
    int64_t B = 1, T = 1, stride_b = 0, stride_t = 0;
    int bytes = 0;
    bool ok = false;
    explicit Tokens(const Tensor* t) {
        if (!t || !t->is_cuda() || !plain(*t)) return;
        bytes = t->scalar_type() == at::kLong ? 8 : t->scalar_type() == at::kInt ? 4 : 0;
        const int64_t dims = t->dim();
        if (dims == 1) {
            T = t->size(0), stride_t = t->stride(0);
        } else if (dims == 2) {
            B = t->size(0), T = t->size(1), stride_b = t->stride(0), stride_t = t->stride(1);
        } else if (dims > 2) {
            return;
        }
        ok = bytes && B <= INT32_MAX && T <= INT32_MAX && B * T < 1 << 26;
    }
};

// embed_forward(forward, stream, tokens, table, scale, dtype)
PyObject* embed_forward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t call_at = in.integer(), stream = in.integer();
    const Tensor *tokens = in.tensor(), *table = in.tensor();
    const double scale = in.number();
    const int64_t out_code = in.integer();
    if (!in.ok || !table || table->dim() != 2 || !table->is_cuda() || out_code < 0) Py_RETURN_NONE;
    const Tokens of(tokens);
    const int code = dtype_code(table->scalar_type());
    const int64_t V = table->size(0), D = table->size(1);
    if (!of.ok || code < 0 || tokens->device() != table->device() || !like(table, *table) || V < 1 ||
        V > HSN_EMBED_MAX_TOKENS || D < 1 || D > HSN_EMBED_MAX_WIDTH)
        Py_RETURN_NONE;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(table->device());
    std::vector<int64_t> shape = tokens->sizes().vec();
    shape.push_back(D);
    const auto type = out_code == 0 ? at::kFloat : out_code == 1 ? at::kHalf : at::kBFloat16;
    const Tensor out = at::empty(shape, at::TensorOptions().device(table->device()).dtype(type));
    const int status = entry<int (*)(P, int64_t, int64_t, int, P, int64_t, int, float, P, int, int, int, int,
                                     int, P)>(call_at)(
        tokens->data_ptr(), of.stride_b, of.stride_t, of.bytes, table->data_ptr(), table->stride(0), code,
        static_cast<float>(scale), out.data_ptr(), out_code, of.B, of.T, V, D, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// embed_backward(workspace, backward, stream, tokens, d_out, V, scale, dtype)
PyObject* embed_backward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *tokens = in.tensor(), *d_out = in.tensor();
    const int64_t V = in.integer();
    const double scale = in.number();
    const int64_t out_code = in.integer();
    if (!in.ok || !d_out || !d_out->is_cuda() || out_code < 0) Py_RETURN_NONE;
    const Tokens of(tokens);
    const int code = dtype_code(d_out->scalar_type());
    if (!of.ok || code < 0 || tokens->device() != d_out->device() || d_out->dim() != tokens->dim() + 1 ||
        !like(d_out, *d_out) || V < 1 || V > HSN_EMBED_MAX_TOKENS)
        Py_RETURN_NONE;
    for (int64_t d = 0; d < tokens->dim(); ++d)
        if (tokens->size(d) != d_out->size(d)) Py_RETURN_NONE;
    const int64_t D = d_out->size(-1), dims = tokens->dim();
    if (D < 1 || D > HSN_EMBED_MAX_WIDTH) Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int, int, int64_t*)>(size_at)(of.B, of.T, V, D, code, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(d_out->device());
    const auto on = at::TensorOptions().device(d_out->device());
    const auto type = out_code == 0 ? at::kFloat : out_code == 1 ? at::kHalf : at::kBFloat16;
    const Tensor d_table = at::empty({V, D}, on.dtype(type));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int64_t, int, P, int64_t, int64_t, int, float, P, int, int, int, int,
                           int, P, int64_t, P)>(call_at)(
        tokens->data_ptr(), of.stride_b, of.stride_t, of.bytes, d_out->data_ptr(),
        dims == 2 ? d_out->stride(0) : 0, dims ? d_out->stride(dims - 1) : 0, code, static_cast<float>(scale),
        d_table.data_ptr(), out_code, of.B, of.T, V, D, ws.data_ptr(), bytes, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(d_table);
    END_HANDLE_TH_ERRORS
}

// Logits [n, V] whose rows are contiguous, and a token a row (int64 or int32).
struct Rows {
    const Tensor *logits, *tokens;
    int code = -1, token_bytes = 0;
    int64_t n = 0, V = 0;
    bool ok = false;
    Rows(const Tensor* l, const Tensor* t) : logits(l), tokens(t) {
        if (!l || !t || l->dim() != 2 || !l->is_cuda()) return;
        code = dtype_code(l->scalar_type());
        n = l->size(0), V = l->size(1);
        token_bytes = t->scalar_type() == at::kLong ? 8 : t->scalar_type() == at::kInt ? 4 : 0;
        ok = code >= 0 && token_bytes && V >= 1 && V <= HSN_SCORE_MAX_TOKENS && n < 1 << 24 &&
             n * V < int64_t(1) << 40 && like(l, *l) && t->dim() == 1 && t->size(0) == n &&
             t->device() == l->device() && plain(*t);
    }
};

// score_forward(workspace, forward, stream, logits, tokens, top, save)
PyObject* score_forward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor *logits = in.tensor(), *tokens = in.tensor();
    const int64_t top = in.integer(), save = in.integer();
    if (!in.ok || top < 0 || top > HSN_SCORE_MAX_TOP) Py_RETURN_NONE;
    const Rows rows(logits, tokens);
    if (!rows.ok) Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int, int64_t*)>(size_at)(rows.n, rows.V, rows.code, top, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(logits->device());
    const auto on = at::TensorOptions().device(logits->device());
    const Tensor logprob = at::empty({rows.n}, on.dtype(at::kFloat));
    const Tensor entropy = at::empty({rows.n}, on.dtype(at::kFloat));
    Tensor top_tokens, top_logprobs, stats;
    if (top) {
        top_tokens = at::empty({rows.n, top}, on.dtype(at::kLong));
        top_logprobs = at::empty({rows.n, top}, on.dtype(at::kFloat));
    }
    if (save) stats = at::empty({rows.n, 4}, on.dtype(at::kFloat));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int, P, int64_t, int, P, P, P, P, P, int, int, int, P, int64_t, P)>(
        call_at)(logits->data_ptr(), logits->stride(0), rows.code, tokens->data_ptr(), tokens->stride(0),
                 rows.token_bytes, logprob.data_ptr(), entropy.data_ptr(),
                 top ? top_tokens.data_ptr() : nullptr, top ? top_logprobs.data_ptr() : nullptr,
                 save ? stats.data_ptr() : nullptr, rows.n, rows.V, top, bytes ? ws.data_ptr() : nullptr, bytes,
                 entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return Py_BuildValue("(NNNNN)", wrap(logprob), wrap(entropy), wrap(top_tokens), wrap(top_logprobs),
                         wrap(stats));
    END_HANDLE_TH_ERRORS
}

// score_backward(backward, stream, logits, tokens, stats, d_logprob, d_entropy)
PyObject* score_backward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t call_at = in.integer(), stream = in.integer();
    const Tensor *logits = in.tensor(), *tokens = in.tensor(), *stats = in.tensor();
    const Tensor *g = in.tensor(), *h = in.tensor();
    if (!in.ok || !stats) Py_RETURN_NONE;
    const Rows rows(logits, tokens);
    if (!rows.ok || !dense(stats, {rows.n, 4}, at::kFloat, logits->device())) Py_RETURN_NONE;
    for (const Tensor* t : {g, h})
        if (t && (t->dim() != 1 || t->size(0) != rows.n || t->scalar_type() != at::kFloat ||
                  t->device() != logits->device() || !plain(*t)))
            Py_RETURN_NONE;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(logits->device());
    const Tensor d = at::empty({rows.n, rows.V},
                               at::TensorOptions().device(logits->device()).dtype(logits->scalar_type()));
    const int status =
        entry<int (*)(P, int64_t, int, P, int64_t, int, P, P, int64_t, P, int64_t, P, int, int, P)>(call_at)(
            logits->data_ptr(), logits->stride(0), rows.code, tokens->data_ptr(), tokens->stride(0),
            rows.token_bytes, stats->data_ptr(), address(g), g ? g->stride(0) : 0, address(h),
            h ? h->stride(0) : 0, d.data_ptr(), rows.n, rows.V, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(d);
    END_HANDLE_TH_ERRORS
}

// unit_router_forward(workspace, forward, stream, logits, k, valid)
PyObject* unit_router_forward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const Tensor* logits = in.tensor();
    const int64_t k = in.integer();
    const Tensor* valid = in.tensor();
    if (!in.ok || !logits || logits->dim() != 2 || !logits->is_cuda()) Py_RETURN_NONE;
    const auto device = logits->device();
    const int code = dtype_code(logits->scalar_type());
    const int64_t n = logits->size(0), M = logits->size(1);
    if (code < 0 || n >= 1 << 30 || M < 1 || M > HSN_ROUTER_MAX_UNITS || k < 1 || k > M ||
        k > HSN_ROUTER_MAX_CHOSEN || !like(logits, *logits) || !dense(valid, {n}, at::kBool, device))
        Py_RETURN_NONE;
    int64_t bytes = 0;
    int status = entry<int (*)(int, int, int, int64_t*)>(size_at)(n, M, code, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(device);
    const auto on = at::TensorOptions().device(device);
    const Tensor units = at::empty({n, k}, on.dtype(at::kLong));
    const Tensor shares = at::empty({n, k}, on.dtype(at::kFloat));
    const Tensor tally = at::empty({M + 1}, on.dtype(at::kLong));
    const Tensor probs = at::empty({M}, on.dtype(at::kFloat));
    const Tensor balance = at::empty({}, on.dtype(at::kFloat));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(P, int64_t, int, P, P, P, P, P, P, int, int, int, P, int64_t, P)>(call_at)(
        logits->data_ptr(), logits->stride(0), code, address(valid), units.data_ptr(), shares.data_ptr(),
        tally.data_ptr(), probs.data_ptr(), balance.data_ptr(), n, M, k, ws.data_ptr(), bytes,
        entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return Py_BuildValue("(NNNNNN)", wrap(units), wrap(shares), wrap(balance), wrap(tally.narrow(0, 0, M)),
                         wrap(probs), wrap(tally));
    END_HANDLE_TH_ERRORS
}

// unit_router_backward(backward, stream, logits, units, tally, d_shares, d_balance, valid)
PyObject* unit_router_backward(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t call_at = in.integer(), stream = in.integer();
    const Tensor *logits = in.tensor(), *units = in.tensor(), *tally = in.tensor();
    const Tensor *g = in.tensor(), *d_balance = in.tensor(), *valid = in.tensor();
    if (!in.ok || !logits || !units || !tally || logits->dim() != 2 || units->dim() != 2 || !logits->is_cuda())
        Py_RETURN_NONE;
    const auto device = logits->device();
    const int code = dtype_code(logits->scalar_type());
    const int64_t n = logits->size(0), M = logits->size(1), k = units->size(1);
    if (code < 0 || n >= 1 << 30 || M < 1 || M > HSN_ROUTER_MAX_UNITS || k < 1 || k > M ||
        k > HSN_ROUTER_MAX_CHOSEN || !like(logits, *logits) || !dense(valid, {n}, at::kBool, device) ||
        !dense(units, {n, k}, at::kLong, device) || !dense(tally, {M + 1}, at::kLong, device))
        Py_RETURN_NONE;
    if (g && (g->dim() != 2 || g->size(0) != n || g->size(1) != k || g->scalar_type() != at::kFloat ||
              g->device() != device || !plain(*g) || (g->stride(1) != 1 && k > 1)))
        Py_RETURN_NONE;
    if (d_balance && (d_balance->numel() != 1 || d_balance->scalar_type() != at::kFloat ||
                      d_balance->device() != device || !plain(*d_balance)))
        Py_RETURN_NONE;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(device);
    const Tensor d = at::empty({n, M}, at::TensorOptions().device(device).dtype(logits->scalar_type()));
    const int status =
        entry<int (*)(P, int64_t, int, P, P, P, P, int64_t, P, P, int, int, int, P)>(call_at)(
            logits->data_ptr(), logits->stride(0), code, address(valid), units->data_ptr(), tally->data_ptr(),
            address(g), g ? g->stride(0) : 0, address(d_balance), d.data_ptr(), n, M, k, entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    return wrap(d);
    END_HANDLE_TH_ERRORS
}

// A list or tuple of tensors, held while it is read.
struct List {
    PyObject* seq = nullptr;
    explicit List(PyObject* o) : seq(PyList_Check(o) || PyTuple_Check(o) ? Py_NewRef(o) : nullptr) {}
    List(const List&) = delete;
    List& operator=(const List&) = delete;
    ~List() { Py_XDECREF(seq); }
    Py_ssize_t size() const { return seq ? PySequence_Fast_GET_SIZE(seq) : 0; }
    const Tensor* at(Py_ssize_t i) const {
        PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
        const bool exact = reinterpret_cast<PyObject*>(Py_TYPE(o)) == THPVariableClass;  // (the usual case)
        return exact || THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
    }
};

// data_ptr() of a tensor that has a storage, inlined: a list has hundreds of them.
void* address_of(const at::TensorImpl* t) {
    char* const base = static_cast<char*>(t->unsafe_storage().unsafeGetStorageImpl()->mutable_data());
    return base + t->storage_offset() * t->itemsize();
}

// grad_clip(workspace, clip, stream, grads, outs, max_norm): outs None: the norm and the coefficient alone
PyObject* grad_clip(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    Arguments in{args, args + n_args};
    const int64_t size_at = in.integer(), call_at = in.integer(), stream = in.integer();
    const List grads(in.next());
    PyObject* const outs_given = in.next();
    const List outs(outs_given);
    const double max_norm = in.number();
    const Py_ssize_t n = grads.size();
    const bool writes = outs_given != Py_None;
    if (!in.ok || n < 1 || n > INT32_MAX || (writes && outs.size() != n) || !(max_norm >= 0.0))
        Py_RETURN_NONE;
    std::vector<void*> at(static_cast<size_t>(2 * n));
    std::vector<int64_t> numels(static_cast<size_t>(n));
    std::vector<int> codes(static_cast<size_t>(n));
    const Tensor* first = grads.at(0);
    if (!first || !first->is_cuda()) Py_RETURN_NONE;
    const auto device = first->device();
    const bool recording = at::GradMode::is_enabled(), in_place = outs_given == grads.seq;
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor* given = grads.at(i);
        if (!given || !plain(*given) || (recording && given->requires_grad())) Py_RETURN_NONE;
        const at::TensorImpl* g = given->unsafeGetTensorImpl();
        codes[i] = dtype_code(given->scalar_type());
        if (codes[i] < 0 || g->device() != device || !g->is_non_overlapping_and_dense()) Py_RETURN_NONE;
        numels[i] = g->numel();
        at[i] = address_of(g);
        if (!writes) continue;
        if (in_place) {
            at[n + i] = at[i];
            continue;
        }
        const Tensor* out = outs.at(i);
        if (!out || !plain(*out) || (recording && out->requires_grad())) Py_RETURN_NONE;
        const at::TensorImpl* o = out->unsafeGetTensorImpl();
        const at::IntArrayRef sizes = g->sizes(), strides = g->strides(), others = o->strides();
        if (out->scalar_type() != given->scalar_type() || o->device() != device || o->sizes() != sizes)
            Py_RETURN_NONE;
        for (size_t d = 0; numels[i] && d < sizes.size(); ++d)
            if (sizes[d] > 1 && others[d] != strides[d]) Py_RETURN_NONE;
        at[n + i] = address_of(o);
    }
    int64_t bytes = 0;
    int status = entry<int (*)(const int64_t*, int, int64_t*)>(size_at)(numels.data(), n, &bytes);
    if (status) return PyLong_FromLong(status);
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard current(device);
    const auto on = at::TensorOptions().device(device);
    const Tensor result = at::empty({2}, on.dtype(at::kDouble));
    const Tensor ws = workspace(bytes, on);
    status = entry<int (*)(void* const*, void* const*, const int64_t*, const int*, int, double, P, P, int64_t,
                           P)>(call_at)(at.data(), writes ? at.data() + n : nullptr, numels.data(),
                                        codes.data(), n, max_norm, result.data_ptr(), ws.data_ptr(), bytes,
                                        entry<P>(stream));
    if (status) return PyLong_FromLong(status);
    for (Py_ssize_t i = 0; writes && i < n; ++i) {  // an update in place, as autograd sees it
        at::TensorImpl* o = outs.at(i)->unsafeGetTensorImpl();
        if (!o->is_inference()) o->bump_version();
    }
    return Py_BuildValue("(NN)", wrap(result.narrow(0, 0, 1)), wrap(result.narrow(0, 1, 1)));
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
    {"embed_forward", fast<embed_forward>(), METH_FASTCALL,
     "(forward, stream, tokens, table, scale, dtype) -> out"},
    {"embed_backward", fast<embed_backward>(), METH_FASTCALL,
     "(workspace, backward, stream, tokens, d_out, V, scale, dtype) -> d_table"},
    {"score_forward", fast<score_forward>(), METH_FASTCALL,
     "(workspace, forward, stream, logits, tokens, top, save) -> (logprob, entropy, top_tokens, "
     "top_logprobs, stats)"},
    {"score_backward", fast<score_backward>(), METH_FASTCALL,
     "(backward, stream, logits, tokens, stats, d_logprob, d_entropy) -> d_logits"},
    {"unit_router_forward", fast<unit_router_forward>(), METH_FASTCALL,
     "(workspace, forward, stream, logits, k, valid) -> (units, shares, balance, counts, probs, tally)"},
    {"unit_router_backward", fast<unit_router_backward>(), METH_FASTCALL,
     "(backward, stream, logits, units, tally, d_shares, d_balance, valid) -> d_logits"},
    {"grad_clip", fast<grad_clip>(), METH_FASTCALL,
     "(workspace, clip, stream, grads, outs, max_norm) -> (norm, coefficient)"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_calls",
                       "The language-model operators' calls in one step (host code only).", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&kModule); }
