// Host side of the adapter operators' usual calls: contiguous tensors of the current device.  On a few rows the GPU is done in
// 3 to 6 us, and checking the arguments in Python and handing them over through ctypes took 9 (route: 12); here it is 4.6 (7.1).
// Each function checks what its Python counterpart in ops.py checks and answers None where anything is not as usual (a view,
// another device, a gradient, a bad argument): the counterpart then takes the call, or says what is wrong with it.  Where the
// dispatcher has more to do than to find the GPU's kernel it answers NotImplemented, before it looks at anything else.  There is
// no kernel here: the entries of include/fr_hip.h are bound by address.
#include <Python.h>

#include <string.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DispatchKeySet.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fr_hip.h"

namespace {

struct Entries {
    decltype(&fr_linear) linear;
    decltype(&fr_linear_workspace_bytes) linear_bytes;
    decltype(&fr_block_norm) block_norm;
    decltype(&fr_route) route;
    decltype(&fr_route_workspace_bytes) route_bytes;
    decltype(&fr_expert_linear) expert_linear;
    decltype(&fr_last_error) last_error;
} entries;

constexpr int64_t INT_END = 1ll << 31;

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return FR_TYPE_F32;
        case at::kBFloat16: return FR_TYPE_BF16;
        case at::kHalf: return FR_TYPE_F16;
        default: return -1;
    }
}

// Whether a tensor is more than memory on one device (a subclass, a negative bit, a batch of a transform, a zero without memory), or
// the thread is in a tracer, a mode or a transform that has to see the operator.  The key sets of both say so; the keys of a plain
// call are those of a backend, of autograd (which refuses or does nothing) and of autocast (which has no rule for these operators).
bool interposed(PyObject* const* args, Py_ssize_t count) {
    static const uint64_t plain = c10::full_backend_mask | c10::DispatchKeySet(c10::DispatchKey::Dense).raw_repr() |
                                  c10::autograd_dispatch_keyset_with_ADInplaceOrView.raw_repr() | c10::autocast_dispatch_keyset.raw_repr() |
                                  c10::DispatchKeySet(c10::DispatchKey::BackendSelect).raw_repr();
    const c10::impl::LocalDispatchKeySet thread = c10::impl::tls_local_dispatch_key_set();
    if ((thread.included_.raw_repr() & ~thread.excluded_.raw_repr() & ~plain) || at::impl::torch_function_mode_enabled()) return true;
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* a = args[i];
        if (a == Py_None || PyLong_Check(a) || PyFloat_Check(a) || THPDtype_Check(a) || !THPVariable_Check(a)) continue;     // the last one is slow for these
        if (!THPVariable_CheckExact(a) || (THPVariable_Unpack(a).key_set().raw_repr() & ~plain)) return true;
    }
    return false;
}

// The arguments of a call.  `usual` turns false at the first that is not.
struct Call {
    PyObject* const* args;
    int device;
    bool usual = true, graded = false;

    // A tensor (NULL for None) that is plain, contiguous and on the device.
    const at::Tensor* tensor(int i) {
        if (args[i] == Py_None) return nullptr;
        if (!THPVariable_CheckExact(args[i])) { usual = false; return nullptr; }
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.get_device() != device || !t.is_contiguous() ||
            (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined()) {
            usual = false;
            return nullptr;
        }
        return &t;
    }
    const at::Tensor* needed(int i) {
        const at::Tensor* t = tensor(i);
        if (!t) usual = false;
        return t;
    }
    int64_t whole(int i) {
        const long long v = PyLong_CheckExact(args[i]) || PyBool_Check(args[i]) ? PyLong_AsLongLong(args[i]) : -1;
        if (v < 0) { PyErr_Clear(); usual = false; }         // no argument here is negative
        return v;
    }
    float real(int i) {
        if (PyFloat_CheckExact(args[i])) return (float)PyFloat_AS_DOUBLE(args[i]);
        if (PyLong_CheckExact(args[i])) {
            const double v = PyLong_AsDouble(args[i]);
            if (!PyErr_Occurred()) return (float)v;
            PyErr_Clear();
        }
        usual = false;
        return 0.f;
    }
    at::ScalarType dtype(int i, at::ScalarType otherwise) {
        if (args[i] == Py_None) return otherwise;
        if (!THPDtype_Check(args[i])) { usual = false; return otherwise; }
        return reinterpret_cast<THPDtype*>(args[i])->scalar_type;
    }
    bool vector(const at::Tensor* t, int64_t n, at::ScalarType also) {       // absent, or [n] of f32 or `also`
        return !t || (t->dim() == 1 && t->size(0) == n && (t->scalar_type() == at::kFloat || t->scalar_type() == also));
    }
};

const void* at_of(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }
const float* floats(const at::Tensor* t) { return static_cast<const float*>(at_of(t)); }
int type_or(const at::Tensor* t, int otherwise) { return t ? type_of(t->scalar_type()) : otherwise; }

struct WithoutGil {                                          // allocations and launches may wait for the GPU
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

at::Tensor make(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
    at::AutoDispatchBelowADInplaceOrView below;
    return at::empty(shape, like.options().dtype(type));
}

PyObject* failed(const char* name, int rc) {
    const char* what = entries.last_error();
    return PyErr_Format(PyExc_RuntimeError, "%s failed (fr_status %d): %s", name, rc, what ? what : "");
}

#define USUAL(ok) do { if (!(ok)) Py_RETURN_NONE; } while (0)
#define ARGUMENTS(n) do { if (count != (n)) return PyErr_Format(PyExc_TypeError, "%d arguments expected", n); } while (0)
#define DIRECT() do { if (interposed(args, count)) Py_RETURN_NOTIMPLEMENTED; } while (0)

// linear(x, weight, bias, slope, residual, act, out_dtype, device, stream)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGUMENTS(9);
    DIRECT();
    Call c{args, (int)PyLong_AsLong(args[7])};
    void* stream = PyLong_AsVoidPtr(args[8]);
    const at::Tensor *x = c.needed(0), *w = c.needed(1), *bias = c.tensor(2), *slope = c.tensor(3), *res = c.tensor(4);
    const int64_t act = c.whole(5);
    USUAL(c.usual && x->dim() >= 1 && w->dim() == 2);
    const int64_t N = w->size(0), K = w->size(1);
    const at::ScalarType type = x->scalar_type(), out_type = c.dtype(6, type);
    USUAL(c.usual && N >= 1 && K >= 1 && N < INT_END && K < INT_END && x->sizes().back() == K && x->numel() > 0);
    USUAL(type_of(type) >= 0 && type_of(out_type) >= 0 && w->scalar_type() == type);
    USUAL(c.vector(bias, N, type) && c.vector(slope, N, at::kFloat) && (slope != nullptr) == (act == FR_ACT_PRELU));
    c10::DimVector shape(x->sizes());
    shape.back() = N;
    USUAL(!res || (res->sizes() == at::IntArrayRef(shape) && type_of(res->scalar_type()) >= 0));
    const int64_t M = x->numel() / K;
    const int kind = type_of(type);
    size_t need = 0;
    int rc;
    at::Tensor out, scratch;
    {
        WithoutGil released;
        rc = entries.linear_bytes(M, (int)N, (int)K, kind, &need);
        if (!rc) {
            out = make(*x, shape, out_type);
            if (need) scratch = make(*x, (int64_t)need, at::kByte);
            rc = entries.linear(x->const_data_ptr(), K, w->const_data_ptr(), at_of(bias), floats(slope), at_of(res), res ? N : 0, out.mutable_data_ptr(),
                                M, (int)N, (int)K, kind, type_or(bias, kind), type_or(res, kind), type_of(out_type), (int)act,
                                need ? scratch.mutable_data_ptr() : nullptr, need, stream);
        }
    }
    return rc ? failed("fr_linear", rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// block_norm(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm, next_weight, next_bias,
//            next_eps, out_dtype, next_dtype, device, stream) -> (out, next or None)
PyObject* block_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGUMENTS(18);
    DIRECT();
    Call c{args, (int)PyLong_AsLong(args[16])};
    void* stream = PyLong_AsVoidPtr(args[17]);
    const at::Tensor *x = c.needed(0), *res = c.tensor(1), *slots = c.tensor(2), *w = c.tensor(4), *b = c.tensor(5), *gate = c.tensor(7),
                     *nw = c.tensor(11), *nb = c.tensor(12);
    const int64_t norm = c.whole(3), gate_act = c.whole(8), next = c.whole(10);
    const float eps = c.real(6), scale = c.real(9), next_eps = c.real(13);
    USUAL(c.usual && x->dim() >= (slots ? 2 : 1) && x->numel() > 0);
    const at::ScalarType out_type = c.dtype(14, x->scalar_type()), next_type = c.dtype(15, out_type);
    const int64_t d = x->sizes().back();
    USUAL(c.usual && d <= 16384 && type_of(x->scalar_type()) >= 0 && type_of(out_type) >= 0 && type_of(next_type) >= 0);
    c10::DimVector shape(x->sizes());
    int64_t S = 0;
    if (slots) {
        shape.pop_back();
        USUAL(slots->sizes() == at::IntArrayRef(shape) && slots->scalar_type() == at::kFloat);
        S = shape.back();
        shape.back() = d;
        USUAL(S < INT_END);
    }
    const bool affine = norm == FR_NORM_RMS || norm == FR_NORM_LAYER, next_affine = next == FR_NORM_RMS || next == FR_NORM_LAYER;
    USUAL((affine || (!w && !b)) && (next_affine || (!nw && !nb)));
    USUAL(c.vector(w, d, at::kFloat) && c.vector(b, d, at::kFloat) && c.vector(nw, d, at::kFloat) && c.vector(nb, d, at::kFloat));
    USUAL(!res || (res->sizes() == at::IntArrayRef(shape) && type_of(res->scalar_type()) >= 0));
    int64_t ldt = 0;
    int ldc = 0;
    if (gate) {
        USUAL(type_of(gate->scalar_type()) >= 0);
        if (gate->dim() == 1 && gate->size(0) == d) ldc = 1;
        else if (gate->sizes() == at::IntArrayRef(shape)) { ldt = d; ldc = 1; }
        else {
            c10::DimVector column(shape);
            column.back() = 1;
            USUAL(gate->sizes() == at::IntArrayRef(column));
            ldt = 1;
        }
    }
    int rc;
    at::Tensor out, nxt;
    {
        WithoutGil released;
        out = make(*x, shape, out_type);
        if (next) nxt = make(*x, shape, next_type);
        rc = entries.block_norm(x->const_data_ptr(), type_of(x->scalar_type()), (int)S, floats(slots), out.numel() / d, (int)d, (int)norm, floats(w), floats(b), eps,
                                at_of(gate), type_or(gate, 0), ldt, ldc, (int)gate_act, scale, at_of(res), type_or(res, 0), out.mutable_data_ptr(), type_of(out_type),
                                (int)next, floats(nw), floats(nb), next_eps, next ? nxt.mutable_data_ptr() : nullptr, type_of(next_type), stream);
    }
    if (rc) return failed("fr_block_norm", rc);
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(out)));
    if (!next) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(both, 1, next ? THPVariable_Wrap(std::move(nxt)) : Py_None);
    return both;
    END_HANDLE_TH_ERRORS
}

// route(logits, k, score, bias, groups, top_groups, renormalise, scale, device, stream) -> (weights, experts, order, offsets)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGUMENTS(10);
    DIRECT();
    Call c{args, (int)PyLong_AsLong(args[8])};
    void* stream = PyLong_AsVoidPtr(args[9]);
    const at::Tensor *logits = c.needed(0), *bias = c.tensor(3);
    const int64_t k = c.whole(1), score = c.whole(2), groups = c.whole(4), top = c.whole(5), renormalise = c.whole(6);
    const float scale = c.real(7);
    USUAL(c.usual && logits->dim() == 2 && type_of(logits->scalar_type()) >= 0);
    const int64_t T = logits->size(0), E = logits->size(1);
    USUAL(E >= 1 && E <= 512 && k >= 1 && k <= 16 && k <= E && groups >= 1 && groups <= 64 && top >= 1 && top <= groups && c.vector(bias, E, at::kFloat));
    size_t need = 0;
    int rc;
    at::Tensor out[4], scratch;
    {
        WithoutGil released;
        rc = entries.route_bytes(T, (int)E, (int)k, &need);
        if (!rc) {
            out[0] = make(*logits, {T, k}, at::kFloat);
            out[1] = make(*logits, {T, k}, at::kInt);
            out[2] = make(*logits, T * k, at::kInt);
            out[3] = make(*logits, E + 1, at::kInt);
            if (need) scratch = make(*logits, (int64_t)need, at::kByte);
            rc = entries.route(logits->const_data_ptr(), type_of(logits->scalar_type()), T, (int)E, (int)k, (int)score, floats(bias), (int)groups, (int)top,
                               renormalise != 0, scale, static_cast<float*>(out[0].mutable_data_ptr()), static_cast<int32_t*>(out[1].mutable_data_ptr()),
                               static_cast<int32_t*>(out[2].mutable_data_ptr()), static_cast<int32_t*>(out[3].mutable_data_ptr()),
                               need ? scratch.mutable_data_ptr() : nullptr, need, stream);
        }
    }
    if (rc) return failed("fr_route", rc);
    PyObject* all = PyTuple_New(4);
    if (!all) return nullptr;
    for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(all, i, THPVariable_Wrap(std::move(out[i])));
    return all;
    END_HANDLE_TH_ERRORS
}

// expert_linear(x, weight, order, offsets, k, bias, act, slope, rows_sorted, out_slots, out_dtype, device, stream)
PyObject* expert_linear(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    ARGUMENTS(13);
    DIRECT();
    Call c{args, (int)PyLong_AsLong(args[11])};
    void* stream = PyLong_AsVoidPtr(args[12]);
    const at::Tensor *x = c.needed(0), *w = c.needed(1), *order = c.needed(2), *offsets = c.needed(3), *bias = c.tensor(5), *slope = c.tensor(7);
    const int64_t k = c.whole(4), act = c.whole(6), rows_sorted = c.whole(8), out_slots = c.whole(9);
    USUAL(c.usual && x->dim() == 2 && w->dim() == 3 && order->dim() == 1 && offsets->dim() == 1);
    const int64_t E = w->size(0), N = w->size(1), K = w->size(2), P = order->size(0);
    const at::ScalarType type = x->scalar_type(), out_type = c.dtype(10, type);
    USUAL(c.usual && E >= 1 && N >= 1 && K >= 1 && E < INT_END && N < INT_END && K < INT_END && x->size(1) == K);
    USUAL(order->scalar_type() == at::kInt && offsets->scalar_type() == at::kInt && offsets->size(0) == E + 1);
    USUAL(k >= 1 && P > 0 && P < INT_END && P % k == 0 && x->size(0) == (rows_sorted ? P : P / k));
    USUAL(type_of(type) >= 0 && type_of(out_type) >= 0 && w->scalar_type() == type && (slope != nullptr) == (act == FR_ACT_PRELU));
    for (const at::Tensor* t : {bias, slope}) USUAL(!t || (t->dim() == 2 && t->size(0) == E && t->size(1) == N));
    USUAL(!bias || bias->scalar_type() == type || bias->scalar_type() == at::kFloat);
    USUAL(!slope || slope->scalar_type() == at::kFloat);
    const int kind = type_of(type);
    int rc;
    at::Tensor out;
    {
        WithoutGil released;
        out = out_slots ? make(*x, {P / k, k, N}, out_type) : make(*x, {P, N}, out_type);
        rc = entries.expert_linear(x->const_data_ptr(), rows_sorted != 0, w->const_data_ptr(), at_of(bias), floats(slope),
                                   static_cast<const int32_t*>(order->const_data_ptr()), static_cast<const int32_t*>(offsets->const_data_ptr()),
                                   out.mutable_data_ptr(), out_slots != 0, P / k, (int)k, (int)E, (int)N, (int)K, kind, type_or(bias, kind), type_of(out_type),
                                   (int)act, stream);
    }
    return rc ? failed("fr_expert_linear", rc) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(addresses of the entries, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
    void* at[sizeof(Entries) / sizeof(void*)];
    ARGUMENTS((int)(sizeof at / sizeof at[0]));
    for (Py_ssize_t i = 0; i < count; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    memcpy(&entries, at, sizeof at);
    Py_RETURN_NONE;
}

#define ENTRY(name) {#name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(linear), ENTRY(block_norm), ENTRY(route), ENTRY(expert_linear), ENTRY(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fr_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fr_calls() { return PyModule_Create(&module); }
