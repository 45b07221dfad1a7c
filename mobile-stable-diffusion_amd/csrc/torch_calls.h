// What the native calls of the Python package are made of (torch_calls.cpp, torch_calls_cl_q4.cpp): checks of plain tensors,
// outputs, the current stream, and the binding to the C ABI of the library the package has loaded.  A source file defines
// MSD_CALLS(X), the entry points it calls, and includes this.
//
// Tensors are read through inline accessors, so an extension is good for the one Python and torch it was compiled for:
// `built_for` names them, and the package asks before it makes any other call there.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/msd_hip.h"

namespace {

struct Abi {
#define X(name) decltype(&::name) name = nullptr;
    MSD_CALLS(X)
#undef X
} abi;
PyObject *raise_code = nullptr;  // the package's check(code)

// Gathers what a call is made of; `ok` turns false at the first thing that is not plain.
struct Call {
    bool ok = true;

    Call(Py_ssize_t given, Py_ssize_t wanted) {
        ok = given == wanted && raise_code != nullptr && !at::impl::torch_function_mode_enabled() &&
             !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
             !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
             !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Functionalize) &&
             !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer);
    }
    // A tensor on a device, of torch's own class (or a Parameter).
    const at::Tensor *strided(PyObject *o) {
        if (!ok) return nullptr;
        if (!THPVariable_CheckExact(o)) return fail();
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.defined()) return fail();
        const c10::DispatchKeySet keys = t.key_set();
        constexpr c10::DispatchKeySet kWrapped(
            {c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
             c10::DispatchKey::Python, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
        if (!t.is_cuda() || t.layout() != at::kStrided || keys.has_any(kWrapped) || !t.has_storage()) return fail();
        return &t;
    }
    // ... dense and contiguous.
    const at::Tensor *tensor(PyObject *o) {
        const at::Tensor *t = strided(o);
        return t != nullptr && t->is_contiguous() ? t : fail();
    }
    // ... of float32 or float16; `code` receives which.
    const at::Tensor *data(PyObject *o, int *code) {
        const at::Tensor *t = tensor(o);
        if (t == nullptr) return nullptr;
        if (t->scalar_type() == at::kFloat) *code = MSD_DTYPE_F32;
        else if (t->scalar_type() == at::kHalf) *code = MSD_DTYPE_F16;
        else return fail();
        return t;
    }
    // dtype and device of `like`, `numel` elements
    const at::Tensor *same(PyObject *o, const at::Tensor &like, int64_t numel) {
        const at::Tensor *t = tensor(o);
        if (t == nullptr) return nullptr;
        if (t->scalar_type() != like.scalar_type() || t->get_device() != like.get_device() || t->numel() != numel) return fail();
        return t;
    }
    const float *affine(PyObject *o, int64_t n, const at::Tensor &like) {
        const at::Tensor *t = tensor(o);
        if (t == nullptr) return nullptr;
        if (t->scalar_type() != at::kFloat || t->numel() != n || t->get_device() != like.get_device()) {
            ok = false;
            return nullptr;
        }
        return static_cast<const float *>(t->data_ptr());
    }
    double number(PyObject *o) {
        if (!ok) return 0;
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    int64_t integer(PyObject *o) {
        if (!ok) return 0;
        if (!PyLong_Check(o)) {  // (a bool is one)
            ok = false;
            return 0;
        }
        const long long v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            ok = false;
        }
        return v;
    }
    // a C int; what does not fit one is the general path's to convert or refuse
    int code(PyObject *o) {
        const int64_t v = integer(o);
        if (v != (int)v) ok = false;
        return (int)v;
    }
    int truth(PyObject *o) {
        if (ok && !PyBool_Check(o)) ok = false;
        return o == Py_True;
    }
    const at::Tensor *fail() {
        ok = false;
        return nullptr;
    }
};

// A new tensor on the device of `like`, past the dispatcher, which has nothing to say about plain calls (Call): 0.4 us
// less than at::empty.
at::Tensor new_tensor(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
    return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

// Whether a contiguous tensor has the strides that a new one of its shape gets.  Those of axes of length one can be any
// (channels last with one position per channel), and torch.empty_like keeps them.
bool plain_strides(const at::Tensor &t) {
    const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
    int64_t stride = 1;
    for (size_t i = sizes.size(); i-- > 0; stride *= std::max<int64_t>(sizes[i], 1))
        if (strides[i] != stride) return false;
    return true;
}

// An output: the caller's tensor, or a new one.
struct Out {
    PyObject *object = nullptr;  // the caller's
    at::Tensor fresh;
    void *data = nullptr;

    void take(Call &c, PyObject *o, const at::Tensor &like) {  // like `like`, or what the caller gave
        if (!c.ok) return;
        if (o == Py_None) {
            if (!plain_strides(like)) {
                c.ok = false;
                return;
            }
            make(new_tensor(like.sizes(), like.scalar_type(), like));
        } else if (const at::Tensor *t = c.same(o, like, like.numel())) {
            object = o;
            data = t->data_ptr();
        }
    }
    void make(at::Tensor t) {
        fresh = std::move(t);
        data = fresh.data_ptr();
    }
    PyObject *result() {
        if (object == nullptr) return THPVariable_Wrap(std::move(fresh));
        Py_INCREF(object);
        return object;
    }
};

// The current stream of the current device; the GIL is given up around the call, as ctypes does.
template <typename F>
int on_stream(F f) {
    void *stream = c10::hip::getCurrentHIPStream(c10::hip::current_device()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f(stream);
    Py_END_ALLOW_THREADS
    return rc;
}

// What `body` returns, None where it returns nullptr without an error set, and for C++ exceptions.
template <typename F>
PyObject *plainly(F body) {
    try {
        PyObject *r = body();
        if (r != nullptr || PyErr_Occurred()) return r;
    } catch (...) {
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// nullptr with the package's exception set for a code other than 0
bool failed(int rc) {
    if (rc == 0) return false;
    PyObject *r = PyObject_CallFunction(raise_code, "i", rc);
    if (r != nullptr) {
        Py_DECREF(r);
        PyErr_SetString(PyExc_RuntimeError, "msd call failed");
    }
    return true;
}

PyObject *finish(int rc, Out &out) { return failed(rc) ? nullptr : out.result(); }

typedef PyObject *const *Args;

// bind(addresses by name, check): the library's entry points and what raises their error codes
PyObject *bind(PyObject *, PyObject *args) {
    PyObject *addresses = nullptr, *check = nullptr;
    if (!PyArg_ParseTuple(args, "O!O", &PyDict_Type, &addresses, &check)) return nullptr;
    Abi bound;
#define X(name)                                                                                      \
    {                                                                                                \
        PyObject *at = PyDict_GetItemString(addresses, #name);                                       \
        void *p = at != nullptr ? PyLong_AsVoidPtr(at) : nullptr;                                    \
        if (p == nullptr) {                                                                          \
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #name);                           \
            return nullptr;                                                                          \
        }                                                                                            \
        bound.name = reinterpret_cast<decltype(bound.name)>(p);                                      \
    }
    MSD_CALLS(X)
#undef X
    Py_INCREF(check);
    Py_XDECREF(raise_code);
    raise_code = check;
    abi = bound;
    Py_RETURN_NONE;
}

PyObject *names(PyObject *, PyObject *) {
    PyObject *list = PyList_New(0);
#define X(name)                                                    \
    if (list != nullptr) {                                         \
        PyObject *s = PyUnicode_FromString(#name);                 \
        if (s == nullptr || PyList_Append(list, s) != 0) Py_CLEAR(list); \
        Py_XDECREF(s);                                             \
    }
    MSD_CALLS(X)
#undef X
    return list;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}

PyObject *make_module(PyModuleDef *definition) {
    PyObject *m = PyModule_Create(definition);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", MSD_BUILT_FOR) != 0) Py_CLEAR(m);
    return m;
}

}  // namespace
