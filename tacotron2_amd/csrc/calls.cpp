// The plain case of the calls in inversion.py without the interpreter's share of it: contiguous tensors of one GPU that is the
// current one, results of its own, nothing recorded by autograd.  Every function returns None for anything else, arguments
// that are to be refused among them; inversion.py then checks, copies, refuses and calls by itself.  Small calls are bound by the
// host: dense 1 x 512 -> 1025 11.0 us a call through ctypes, 4.8 here; gradients of 641 x 80 -> 512 21.6 and 10.3.
#include <Python.h>

#include <cmath>
#include <initializer_list>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/gl_hip.h"

namespace {

// The library's entry points, as inversion.py has them loaded
decltype(&gl_dense_workspace) dense_workspace;
decltype(&gl_dense) dense_call;
decltype(&gl_dense_backward_workspace) dense_backward_workspace;
decltype(&gl_dense_backward) dense_backward_call;
decltype(&gl_group_norm_workspace) group_norm_workspace;
decltype(&gl_group_norm) group_norm_call;
decltype(&gl_group_norm_backward_workspace) group_norm_backward_workspace;
decltype(&gl_group_norm_backward) group_norm_backward_call;
PyObject* raw_stream;                    // device index -> the current stream's handle

int type_of(c10::ScalarType t) {
    return t == at::kFloat ? GL_F32 : t == at::kBFloat16 ? GL_BF16 : t == at::kHalf ? GL_F16 : -1;
}

// An argument: absent, a plain tensor, or something this file does not deal with
struct Arg {
    const at::Tensor* t = nullptr;
    bool other = false;
    explicit Arg(PyObject* o) {
        if (o == Py_None) return;
        if (!THPVariable_CheckExact(o) || THPVariable_Unpack(o)._fw_grad(0).defined()) other = true;     // with a tangent: refused
        else t = &THPVariable_Unpack(o);
    }
    explicit operator bool() const { return t; }
    const at::Tensor* operator->() const { return t; }
    void* p() const { return t ? t->data_ptr() : nullptr; }
    // contiguous, of this type on this device, with these sizes; an absent one is plain
    bool plain(c10::ScalarType type, c10::Device device, at::IntArrayRef sizes) const {
        if (!t) return !other;
        return t->layout() == at::kStrided && t->scalar_type() == type && t->device() == device && t->sizes() == sizes && t->is_contiguous();
    }
};

// A first argument that leads: float type, contiguous, on the current device
bool leads(const Arg& x) {
    if (torch::jit::tracer::isTracing()) return false;       // refused
    if (!x || x->layout() != at::kStrided || !x->is_cuda() || x->dim() < 1 || x->numel() == 0 || !x->is_contiguous()) return false;
    if (type_of(x->scalar_type()) < 0) return false;
    return c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice() == x->device();
}
bool recorded(std::initializer_list<const Arg*> args) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const Arg* a : args)
        if (*a && (*a)->requires_grad()) return true;
    return false;
}
bool apart(const at::Tensor& out, std::initializer_list<const Arg*> args) {
    const char *a0 = (const char*)out.data_ptr(), *a1 = a0 + out.nbytes();
    for (const Arg* a : args)
        if (*a) {
            const char* b0 = (const char*)a->p();
            if (a0 < b0 + (*a)->nbytes() && b0 < a1) return false;
        }
    return true;
}

// What a call writes into a tensor of the caller's counts as a change of it: autograd then finds gradients that would be stale
void written(const Arg& a) {
    if (a && !a->is_inference()) a->unsafeGetTensorImpl()->bump_version();
}

at::Tensor scratch(long long bytes, const at::Tensor& like) {
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The current stream of a device; false with a Python error set
bool stream_of(c10::Device device, void** stream) {
    PyObject* index = PyLong_FromLong(device.index());
    if (!index) return false;
    PyObject* handle = PyObject_CallOneArg(raw_stream, index);
    Py_DECREF(index);
    if (!handle) return false;
    *stream = PyLong_AsVoidPtr(handle);
    Py_DECREF(handle);
    return !PyErr_Occurred();
}

// f() with C++ exceptions as the Python errors that torch makes of them (torch.OutOfMemoryError among them); f returns a new
// reference, or null for "not here"
template <typename F>
PyObject* guarded(F f) {
    try {
        PyObject* r = f();
        if (r || PyErr_Occurred()) return r;
        Py_RETURN_NONE;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}
bool numbers(PyObject* const* o, int n, long* v) {           // false with an error set where one is not a number
    for (int k = 0; k < n; ++k) {
        v[k] = PyLong_AsLong(o[k]);
        if (v[k] == -1 && PyErr_Occurred()) return false;
    }
    return true;
}
PyObject* wrap(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}
PyObject* wrap3(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    const at::Tensor* all[3] = {&a, &b, &c};
    for (int k = 0; k < 3; ++k) {
        PyObject* o = wrap(*all[k]);
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, k, o);
    }
    return r;
}

// dense(x, weight, bias, residual, preactivation, out_dtype, act)
PyObject* dense(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 7) return nullptr;
        const Arg x(o[0]), w(o[1]), b(o[2]), r(o[3]), z(o[4]);
        long act;
        if (!numbers(o + 6, 1, &act)) return nullptr;
        if (!leads(x) || !w || w->dim() != 2 || recorded({&x, &w, &b, &r})) return nullptr;
        const auto type = x->scalar_type();
        const auto device = x->device();
        auto to = type;
        if (o[5] != Py_None) {
            if (!THPDtype_Check(o[5])) return nullptr;
            to = ((THPDtype*)o[5])->scalar_type;
            if (to != type && to != at::kFloat) return nullptr;
        }
        const int64_t K = x->size(-1), N = w->size(0), rows = x->numel() / K;
        if (N < 1 || N > 1 << 20 || K > 1 << 20 || rows > 0x7fffffff) return nullptr;
        auto shape = x->sizes().vec();
        shape.back() = N;
        if (!w.plain(type, device, {N, K}) || !b.plain(type, device, {N}) || !r.plain(to, device, shape) || !z.plain(to, device, shape))
            return nullptr;
        if (z && !apart(*z.t, {&x, &w, &b, &r})) return nullptr;
        void* stream;
        if (!stream_of(device, &stream)) return nullptr;
        const at::Tensor y = at::empty(shape, x->options().dtype(to));
        const long long bytes = dense_workspace(rows, (int)K, (int)N, type_of(type), type_of(to));
        const at::Tensor ws = scratch(bytes, *x.t);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = dense_call(x.p(), K, w.p(), K, b.p(), r.p(), N, y.data_ptr(), N, z.p(), N, rows, (int)K, (int)N, type_of(type), type_of(to),
                        (int)act, pointer(ws), bytes, stream);
        Py_END_ALLOW_THREADS
        if (rc) return nullptr;
        written(z);
        return wrap(y);
    });
}

// dense_backward(dy, x, weight, preactivation, act, needs dx, dweight, dbias)
PyObject* dense_backward(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 8) return nullptr;
        const Arg dy(o[0]), x(o[1]), w(o[2]), z(o[3]);
        long v[4];
        if (!numbers(o + 4, 4, v)) return nullptr;
        if (!leads(x) || !dy || !w || w->dim() != 2 || !(v[1] || v[2] || v[3]) || (v[0] && !z)) return nullptr;
        const auto type = x->scalar_type(), from = dy->scalar_type();
        const auto device = x->device();
        if (from != type && from != at::kFloat) return nullptr;
        const int64_t K = x->size(-1), N = w->size(0), rows = x->numel() / K;
        if (N < 1 || N > 1 << 20 || K > 1 << 20 || rows > 0x7fffffff) return nullptr;
        auto shape = x->sizes().vec();
        shape.back() = N;
        if (!w.plain(type, device, {N, K}) || !dy.plain(from, device, shape) || (v[0] && !z.plain(from, device, shape))) return nullptr;
        void* stream;
        if (!stream_of(device, &stream)) return nullptr;
        at::Tensor dx, dw, db;
        if (v[1]) dx = at::empty(x->sizes(), x->options());
        if (v[2]) dw = at::empty({N, K}, x->options());
        if (v[3]) db = at::empty({N}, x->options());
        const long long bytes = dense_backward_workspace(rows, (int)K, (int)N, type_of(type), type_of(from), (int)v[0]);
        const at::Tensor ws = scratch(bytes, *x.t);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = dense_backward_call(dy.p(), N, x.p(), K, w.p(), K, v[0] ? z.p() : nullptr, N, pointer(dx), K, pointer(dw), K, pointer(db), rows,
                                 (int)K, (int)N, type_of(type), type_of(from), (int)v[0], pointer(ws), bytes, stream);
        Py_END_ALLOW_THREADS
        return rc ? nullptr : wrap3(dx, dw, db);
    });
}

struct Frames {                          // (B, T, channels) or (T, channels)
    int64_t B, T, C, G;
    bool of(const at::Tensor& x, long groups) {
        if (x.dim() != 2 && x.dim() != 3) return false;
        B = x.dim() == 2 ? 1 : x.size(0);
        T = x.size(-2);
        C = x.size(-1);
        G = groups;
        return B <= 65535 && T <= 1 << 30 && C <= 1 << 20 && G >= 1 && C % G == 0;
    }
};

// group_norm(x, weight, bias, lengths, stats, groups, act, eps)
PyObject* group_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 8) return nullptr;
        const Arg x(o[0]), w(o[1]), b(o[2]), lens(o[3]), stats(o[4]);
        long v[2];
        if (!numbers(o + 5, 2, v)) return nullptr;
        const double eps = PyFloat_AsDouble(o[7]);
        if (PyErr_Occurred()) return nullptr;
        Frames f;
        if (!leads(x) || recorded({&x, &w, &b}) || !f.of(*x.t, v[0]) || !(eps >= 0)) return nullptr;
        const auto type = x->scalar_type();
        const auto device = x->device();
        if (!w.plain(type, device, {f.C}) || !b.plain(type, device, {f.C}) || !lens.plain(at::kInt, device, {f.B}) ||
            !stats.plain(at::kFloat, device, {f.B, f.G, 2}))
            return nullptr;
        if (stats && !apart(*stats.t, {&x, &w, &b, &lens})) return nullptr;
        void* stream;
        if (!stream_of(device, &stream)) return nullptr;
        const at::Tensor y = at::empty(x->sizes(), x->options());
        const long long bytes = group_norm_workspace((int)f.B, (int)f.T, (int)f.C, (int)f.G, type_of(type));
        const at::Tensor ws = scratch(bytes, *x.t);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = group_norm_call(x.p(), f.C, w.p(), b.p(), (const int*)lens.p(), y.data_ptr(), f.C, (float*)stats.p(), (int)f.B, (int)f.T, (int)f.C,
                             (int)f.G, type_of(type), (int)v[1], (float)eps, pointer(ws), bytes, stream);
        Py_END_ALLOW_THREADS
        if (rc) return nullptr;
        written(stats);
        return wrap(y);
    });
}

// group_norm_backward(dy, x, stats, weight, bias, lengths, groups, act, needs dx, dweight, dbias)
PyObject* group_norm_backward(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 11) return nullptr;
        const Arg dy(o[0]), x(o[1]), stats(o[2]), w(o[3]), b(o[4]), lens(o[5]);
        long v[5];
        if (!numbers(o + 6, 5, v)) return nullptr;
        Frames f;
        if (!leads(x) || !dy || !stats || !f.of(*x.t, v[0])) return nullptr;
        const auto type = x->scalar_type();
        const auto device = x->device();
        if (!dy.plain(type, device, x->sizes()) || !stats.plain(at::kFloat, device, {f.B, f.G, 2}) || !w.plain(type, device, {f.C}) ||
            !b.plain(type, device, {f.C}) || !lens.plain(at::kInt, device, {f.B}))
            return nullptr;
        at::Tensor dx, dw, db;
        if (v[2]) dx = at::empty(x->sizes(), x->options());
        if (v[3] && w) dw = at::empty({f.C}, x->options());
        if (v[4] && b) db = at::empty({f.C}, x->options());
        if (!dx.defined() && !dw.defined() && !db.defined()) return nullptr;
        void* stream;
        if (!stream_of(device, &stream)) return nullptr;
        const long long bytes = group_norm_backward_workspace((int)f.B, (int)f.T, (int)f.C, (int)f.G, type_of(type));
        const at::Tensor ws = scratch(bytes, *x.t);
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = group_norm_backward_call(dy.p(), f.C, x.p(), f.C, (const float*)stats.p(), w.p(), b.p(), (const int*)lens.p(), pointer(dx), f.C,
                                      pointer(dw), pointer(db), (int)f.B, (int)f.T, (int)f.C, (int)f.G, type_of(type), (int)v[1], pointer(ws),
                                      bytes, stream);
        Py_END_ALLOW_THREADS
        return rc ? nullptr : wrap3(dx, dw, db);
    });
}

// bind(raw_stream, the eight addresses in the order of the variables above)
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "bind: nine arguments");
        return nullptr;
    }
    void* p[8];
    for (int k = 0; k < 8; ++k) {
        p[k] = PyLong_AsVoidPtr(o[1 + k]);
        if (PyErr_Occurred()) return nullptr;
    }
    dense_workspace = (decltype(dense_workspace))p[0];
    dense_call = (decltype(dense_call))p[1];
    dense_backward_workspace = (decltype(dense_backward_workspace))p[2];
    dense_backward_call = (decltype(dense_backward_call))p[3];
    group_norm_workspace = (decltype(group_norm_workspace))p[4];
    group_norm_call = (decltype(group_norm_call))p[5];
    group_norm_backward_workspace = (decltype(group_norm_backward_workspace))p[6];
    group_norm_backward_call = (decltype(group_norm_backward_call))p[7];
    Py_XDECREF(raw_stream);
    raw_stream = Py_NewRef(o[0]);
    Py_RETURN_NONE;
}

#define GL_FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {GL_FAST(bind), GL_FAST(dense), GL_FAST(dense_backward), GL_FAST(group_norm), GL_FAST(group_norm_backward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "The plain case of the calls in inversion.py.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
