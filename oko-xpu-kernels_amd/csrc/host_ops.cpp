// The host path of the Python API's hot calls (xpu_kernels.int8 linear, ffn, the
// backward's products and the quantizer; xpu_kernels.mxfp4, moe, norm and rope with their gradients)
// as a CPython extension: argument checks, the packed weight's lookup, allocations and
// the library call in native code.  In Python these cost more than the small calls'
// kernels: linear at 16 x 4096 x 4096 took 17.6 us of host time for 8.5 us of GPU work,
// 6.9 of them the library's two launches.
//
// Every function takes the plain case only -- dense CUDA tensors of exactly the
// dtype, shape, alignment and device the kernels read, no subclass, no
// functorch wrapper, no torch-function or dispatch mode -- and returns None for
// anything else, so that the caller's Python path converts, refuses or computes
// it as before.  Results, and the kernels that run, are the same on both.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Storage.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cstdio>
#include <cstring>
#include <exception>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "xpuint8.h"

namespace {

using at::Tensor;

// ---------------------------------------------------------- the library
// Addresses of the loaded libxpuint8.so's entry points, in the order bind()
// receives them (_lib.py's _HOST_ENTRIES), called by the header's own types.
struct Library {
    decltype(&xpuint8_last_error) last_error;
    decltype(&xpuint8_linear_workspace_size) linear_size;
    decltype(&xpuint8_linear_packed_stream) linear;
    decltype(&xpuint8_ffn_workspace_size) ffn_size;
    decltype(&xpuint8_ffn_packed_stream) ffn;
    decltype(&xpuint8_linear_backward_int8_workspace_size) bwd_int8_size;
    decltype(&xpuint8_linear_backward_int8_stream) bwd_int8;
    decltype(&xpuint8_linear_backward_dense_workspace_size) bwd_dense_size;
    decltype(&xpuint8_linear_backward_dense_stream) bwd_dense;
    decltype(&xpuint8_linear_dx_split_workspace_size) dx_size;
    decltype(&xpuint8_linear_dx_stream) dx;
    decltype(&xpuint8_linear_dw_workspace_size) dw_size;
    decltype(&xpuint8_linear_dw_work_stream) dw;
    decltype(&xpuint8_column_sum_workspace_size) colsum_size;
    decltype(&xpuint8_column_sum_stream) colsum;
    decltype(&xpuint8_convrot_quantize_stream) quantize;
    decltype(&xpuint8_linear_acc_packed_stream) linear_acc;
    decltype(&xpuint8_linear_dx_int8_reads_packed) dx_reads_packed;
    decltype(&xpuint8_mxfp4_quantize_stream) mx_quantize;
    decltype(&xpuint8_mxfp4_dequantize_stream) mx_dequantize;
    decltype(&xpuint8_mxfp4_linear_workspace_size) mx_linear_size;
    decltype(&xpuint8_mxfp4_linear_stream) mx_linear;
    decltype(&xpuint8_mxfp4_grouped_linear_workspace_size) mx_grouped_size;
    decltype(&xpuint8_mxfp4_grouped_linear_stream) mx_grouped;
    decltype(&xpuint8_moe_sort_workspace_size) moe_sort_size;
    decltype(&xpuint8_moe_sort_stream) moe_sort;
    decltype(&xpuint8_moe_dispatch_stream) moe_dispatch;
    decltype(&xpuint8_moe_combine_stream) moe_combine;
    decltype(&xpuint8_mxfp4_dx_workspace_size_of) mx_dx_size;
    decltype(&xpuint8_mxfp4_dx_stream) mx_dx;
    decltype(&xpuint8_moe_combine_grad_stream) moe_combine_grad;
    decltype(&xpuint8_mxfp4_dbias_workspace_size) mx_dbias_size;
    decltype(&xpuint8_mxfp4_dbias_stream) mx_dbias;
    decltype(&xpuint8_rms_norm_stream) rms_norm;
    decltype(&xpuint8_rms_norm_int8_stream) rms_norm_int8;
    decltype(&xpuint8_rms_norm_grad_workspace_size) rms_norm_grad_size;
    decltype(&xpuint8_rms_norm_grad_stream) rms_norm_grad;
    decltype(&xpuint8_rope_axes_stream) rope_axes;
    decltype(&xpuint8_moe_route_stream) moe_route;
    decltype(&xpuint8_moe_route_grad_stream) moe_route_grad;
};
constexpr int kEntries = 40;
static_assert(sizeof(Library) == kEntries * sizeof(void*), "one address per entry");

Library g_lib;
PyObject* g_raw_stream = nullptr;   // device index -> current stream's handle
PyObject* g_capturing = nullptr;    // () -> whether the current stream is being captured
PyObject* g_packed = nullptr;       // the packed-weight registry (ops._PACKED)

// ----------------------------------------------------------- arguments
bool modes_active() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           at::impl::torch_function_mode_enabled();
}

constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper,
                                        c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                        c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                        c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                        c10::DispatchKey::ZeroTensor,
                                        c10::DispatchKey::Batched});

// A plain tensor object's tensor: dense, contiguous, on a GPU, 16-byte aligned
// and not empty; null otherwise.
const Tensor* plain(PyObject* o, at::ScalarType dtype) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || t.scalar_type() != dtype || !t.is_cuda() ||
        t.key_set().has_any(kWrapped) || !t.has_storage() || !t.is_contiguous() ||
        t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)
        return nullptr;
    return &t;
}
// the same, one-dimensional with n values, on the device of `like`
const Tensor* vec(PyObject* o, at::ScalarType dtype, int64_t n, const Tensor& like) {
    const Tensor* t = plain(o, dtype);
    return t && t->dim() == 1 && t->numel() == n && t->device() == like.device() ? t : nullptr;
}
// an int8 [N, K] weight on the device of `like`
const Tensor* weight(PyObject* o, const Tensor& like) {
    const Tensor* t = plain(o, at::kChar);
    return t && t->dim() == 2 && t->device() == like.device() ? t : nullptr;
}

struct Bias {
    bool ok = false;
    const void* p = nullptr;
    int32_t bf16 = 0;
};
Bias bias_arg(PyObject* o, int64_t n, const Tensor& like) {
    Bias b;
    if (o == Py_None) {
        b.ok = true;
    } else if (const Tensor* t = vec(o, at::kBFloat16, n, like)) {
        b = Bias{true, t->data_ptr(), 1};
    } else if (const Tensor* t = vec(o, at::kFloat, n, like)) {
        b = Bias{true, t->data_ptr(), 0};
    }
    return b;
}

// The registry's entry of a weight (a list: weak reference to the storage,
// version, shape, packed copy, second packed form) while it is valid, borrowed;
// null without one.  The rules are ops._packed_entry's.
PyObject* packed_entry(const Tensor& w) {
    if (PyDict_GET_SIZE(g_packed) == 0 || w.is_inference() || w.storage_offset() != 0 ||
        w.size(0) % 16 != 0 || w.size(1) % 16 != 0)
        return nullptr;
    PyObject* key = PyLong_FromVoidPtr(w.storage().mutable_data());
    if (!key) throw python_error();
    PyObject* e = PyDict_GetItemWithError(g_packed, key);   // borrowed
    Py_DECREF(key);
    if (!e) {
        if (PyErr_Occurred()) throw python_error();
        return nullptr;
    }
    if (!PyList_CheckExact(e) || PyList_GET_SIZE(e) != 5) return nullptr;
    PyObject* st = PyWeakref_GetObject(PyList_GET_ITEM(e, 0));     // borrowed
    if (!st || st == Py_None ||
        THPStorage_Unpack(st).unsafeGetStorageImpl() != w.storage().unsafeGetStorageImpl())
        return nullptr;
    PyObject* shape = PyList_GET_ITEM(e, 2);
    if (PyLong_AsLongLong(PyList_GET_ITEM(e, 1)) != int64_t(w._version()) ||
        !PyTuple_CheckExact(shape) || PyTuple_GET_SIZE(shape) != 2 ||
        PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) != w.size(0) ||
        PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 1)) != w.size(1))
        return nullptr;
    return e;
}
// entry e's packed copy (which = 3) or second form (4), undefined for none.  The
// caller holds it until its kernels are enqueued: another thread may pack the
// weight anew, or free it, as soon as the library call lets go of the GIL.
Tensor packed_form(PyObject* e, int which) {
    if (!e) return Tensor();
    PyObject* p = PyList_GET_ITEM(e, which);
    return p == Py_None ? Tensor() : THPVariable_Unpack(p);
}
const int8_t* codes(const Tensor& t) {
    return t.defined() ? static_cast<const int8_t*>(t.data_ptr()) : nullptr;
}

// ------------------------------------------------------------ the call
const void* current_stream(const Tensor& t) {
    PyObject* i = PyLong_FromLong(t.device().index());
    if (!i) throw python_error();
    PyObject* s = PyObject_CallOneArg(g_raw_stream, i);
    Py_DECREF(i);
    if (!s) throw python_error();
    const void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (!p && PyErr_Occurred()) throw python_error();
    return p;
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return at::empty(sizes, at::TensorOptions().dtype(dtype).device(like.device()));
}
Tensor workspace(int64_t bytes, const Tensor& like) { return empty({bytes}, at::kByte, like); }

// RuntimeError(f"{what}: {last_error!r}"), as ops._err raises it
[[noreturn]] void fail(const char* what) {
    PyObject* msg = PyBytes_FromString(g_lib.last_error());
    if (msg) {
        PyErr_Format(PyExc_RuntimeError, "%s: %R", what, msg);
        Py_DECREF(msg);
    }
    throw python_error();
}

// The GIL released for a scope, an exception's way out of it included
struct NoGil {
    PyThreadState* s = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(s); }
};

// f() without the GIL: the allocations (as torch.empty makes them: one that
// misses the allocator's cache can wait for the device) and the library call
// (as ctypes makes it); its error, if any, raised
template <class F>
void call(const char* what, const F& f) {
    int rc;
    {
        NoGil g;
        rc = f();
    }
    if (rc != 0) fail(what);
}

// A Python-callable around f(args): C++ exceptions become Python ones
template <class F>
PyObject* guarded(Py_ssize_t nargs, Py_ssize_t want, const F& f) {
    if (nargs != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, nargs);
        return nullptr;
    }
    try {
        if (!g_raw_stream || !g_packed || modes_active()) Py_RETURN_NONE;
        return f();
    } catch (python_error& e) {
        // raised above with the error indicator set, or carried from torch
        if (!PyErr_Occurred()) e.restore();
        return nullptr;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

PyObject* pair(const Tensor& a, const Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = b.defined() ? THPVariable_Wrap(b) : Py_NewRef(Py_None);
    PyObject* t = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

// x's leading sizes with n for the last
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = n;
    return s;
}

// ------------------------------------------------------------ functions
// linear(x, w8, w_scale, bias): ops.linear without activation or residual
PyObject* host_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 4, [&]() -> PyObject* {
        const Tensor* x = plain(a[0], at::kBFloat16);
        if (!x || x->dim() < 1) Py_RETURN_NONE;
        const Tensor* w = weight(a[1], *x);
        if (!w) Py_RETURN_NONE;
        const int64_t n = w->size(0), k = w->size(1), m = x->numel() / x->size(-1);
        if (x->size(-1) != k || k % 256 != 0 || n % 16 != 0) Py_RETURN_NONE;
        const Tensor* ws = vec(a[2], at::kFloat, n, *x);
        const Bias b = bias_arg(a[3], n, *x);
        if (!ws || !b.ok) Py_RETURN_NONE;
        const int64_t need = g_lib.linear_size(m, n, k);
        if (need < 0) fail("linear");
        const Tensor packed = packed_form(packed_entry(*w), 3);
        const int8_t* p = codes(packed);
        const void* st = current_stream(*x);
        Tensor work, out;
        call("linear", [&] {
            work = workspace(need, *x);
            out = empty(with_last(*x, n), at::kBFloat16, *x);
            return g_lib.linear(st, x->data_ptr(), static_cast<const int8_t*>(w->data_ptr()), p,
                                static_cast<const float*>(ws->data_ptr()), b.p, b.bf16,
                                out.data_ptr(), m, n, k, work.data_ptr(), need);
        });
        return THPVariable_Wrap(out);
    });
}

// linear_acc(x, w8): ops.linear_acc's (int32 [M, N], fp32 [M])
PyObject* host_linear_acc(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject* {
        const Tensor* x = plain(a[0], at::kBFloat16);
        if (!x || x->dim() < 1) Py_RETURN_NONE;
        const Tensor* w = weight(a[1], *x);
        if (!w) Py_RETURN_NONE;
        const int64_t n = w->size(0), k = w->size(1), m = x->numel() / x->size(-1);
        if (x->size(-1) != k || k % 256 != 0 || n % 16 != 0) Py_RETURN_NONE;
        const int64_t need = g_lib.linear_size(m, n, k);
        if (need < 0) fail("linear_acc");
        const Tensor packed = packed_form(packed_entry(*w), 3);
        const int8_t* p = codes(packed);
        const void* st = current_stream(*x);
        Tensor work, acc, xs;
        call("linear_acc", [&] {
            work = workspace(need, *x);
            acc = empty({m, n}, at::kInt, *x);
            xs = empty({m}, at::kFloat, *x);
            return g_lib.linear_acc(st, x->data_ptr(), static_cast<const int8_t*>(w->data_ptr()), p,
                                    static_cast<int32_t*>(acc.data_ptr()),
                                    static_cast<float*>(xs.data_ptr()), m, n, k, work.data_ptr(),
                                    need);
        });
        return pair(acc, xs);
    });
}

// ffn(x, up_w8, up_scale, down_w8, down_scale, down_bias, activation id)
PyObject* host_ffn(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 7, [&]() -> PyObject* {
        const Tensor* x = plain(a[0], at::kBFloat16);
        if (!x || x->dim() < 1) Py_RETURN_NONE;
        const Tensor *up = weight(a[1], *x), *down = weight(a[3], *x);
        if (!up || !down) Py_RETURN_NONE;
        const long act = PyLong_AsLong(a[6]);
        if (act == -1 && PyErr_Occurred()) throw python_error();
        const int64_t n = up->size(0), k = up->size(1), m = x->numel() / x->size(-1);
        const bool paired = act == 3 || act == 4;
        if (!(paired || act == 5) || x->size(-1) != k || k % 256 != 0 || n % 16 != 0 ||
            (paired && n % 2 != 0))
            Py_RETURN_NONE;
        const int64_t inner = paired ? n / 2 : n;
        if (inner % 256 != 0 || down->size(0) != k || down->size(1) != inner) Py_RETURN_NONE;
        const Tensor *us = vec(a[2], at::kFloat, n, *x), *ds = vec(a[4], at::kFloat, k, *x);
        const Bias b = bias_arg(a[5], k, *x);
        if (!us || !ds || !b.ok) Py_RETURN_NONE;
        const int64_t need = g_lib.ffn_size(m, inner, k, int32_t(act));
        if (need < 0) fail("ffn");
        const Tensor up_packed = packed_form(packed_entry(*up), 3),
                     down_packed = packed_form(packed_entry(*down), 3);
        const int8_t *up_p = codes(up_packed), *down_p = codes(down_packed);
        const void* st = current_stream(*x);
        Tensor work, out;
        call("ffn", [&] {
            work = workspace(need, *x);
            out = empty(x->sizes(), at::kBFloat16, *x);
            return g_lib.ffn(st, x->data_ptr(), static_cast<const int8_t*>(up->data_ptr()), up_p,
                             static_cast<const float*>(us->data_ptr()),
                             static_cast<const int8_t*>(down->data_ptr()), down_p,
                             static_cast<const float*>(ds->data_ptr()), b.p, b.bf16, out.data_ptr(),
                             m, inner, k, int32_t(act), work.data_ptr(), need);
        });
        return THPVariable_Wrap(out);
    });
}

// backward(dy, w8, w_scale, want_dbias, dbias_fp32, dense): ops._linear_backward's
// (dx, dbias or None).  The int8 mode of a weight whose second packed form this
// product reads and is still to be made goes through Python, which makes it.
PyObject* host_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 6, [&]() -> PyObject* {
        const Tensor* dy = plain(a[0], at::kBFloat16);
        if (!dy || dy->dim() != 2) Py_RETURN_NONE;
        const Tensor* w = weight(a[1], *dy);
        if (!w) Py_RETURN_NONE;
        const int64_t m = dy->size(0), n = w->size(0), k = w->size(1);
        if (dy->size(1) != n || n % 16 != 0 || k % 256 != 0) Py_RETURN_NONE;
        const Tensor* ws = vec(a[2], at::kFloat, n, *dy);
        if (!ws) Py_RETURN_NONE;
        const int want = PyObject_IsTrue(a[3]), f32 = PyObject_IsTrue(a[4]),
                  dense = PyObject_IsTrue(a[5]);
        if (want < 0 || f32 < 0 || dense < 0) throw python_error();
        const char* what = dense ? "linear_dx" : "linear_dx_int8";
        Tensor packed_nn;
        if (!dense) {
            PyObject* e = packed_entry(*w);
            packed_nn = packed_form(e, 4);
            if (e && !packed_nn.defined() && g_lib.dx_reads_packed(m, n, k) == 1) Py_RETURN_NONE;
        }
        const int8_t* nn = codes(packed_nn);
        const int64_t need = (dense ? g_lib.bwd_dense_size : g_lib.bwd_int8_size)(m, n, k);
        if (need < 0) fail(what);
        const int8_t* wp = static_cast<const int8_t*>(w->data_ptr());
        const float* wsp = static_cast<const float*>(ws->data_ptr());
        const void* st = current_stream(*dy);
        Tensor work, dx, db;
        call(what, [&] {
            work = workspace(need, *dy);
            dx = empty({m, k}, at::kBFloat16, *dy);
            if (want) db = empty({n}, f32 ? at::kFloat : at::kBFloat16, *dy);
            void* dbp = want ? db.data_ptr() : nullptr;
            return dense ? g_lib.bwd_dense(st, dy->data_ptr(), wp, wsp, dx.data_ptr(), dbp,
                                           want && f32, m, n, k, work.data_ptr(), need)
                         : g_lib.bwd_int8(st, dy->data_ptr(), wsp, wp, nn, dx.data_ptr(), dbp,
                                          want && f32, m, n, k, work.data_ptr(), need);
        });
        return pair(dx, db);
    });
}

// linear_dx(dy, w): dy [.., N] @ w [N, K], both bf16
PyObject* host_linear_dx(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject* {
        const Tensor *dy = plain(a[0], at::kBFloat16), *w = plain(a[1], at::kBFloat16);
        if (!dy || !w || dy->dim() < 1 || w->dim() != 2 || w->device() != dy->device())
            Py_RETURN_NONE;
        const int64_t n = w->size(0), k = w->size(1), m = dy->numel() / dy->size(-1);
        if (dy->size(-1) != n || n % 16 != 0 || k % 16 != 0) Py_RETURN_NONE;
        const int64_t need = g_lib.dx_size(m, n, k);
        if (need < 0) fail("linear_dx");
        const void* st = current_stream(*dy);
        Tensor work, dx;
        call("linear_dx", [&] {
            if (need > 0) work = workspace(need, *dy);
            dx = empty(with_last(*dy, k), at::kBFloat16, *dy);
            return g_lib.dx(st, dy->data_ptr(), w->data_ptr(), dx.data_ptr(), m, n, k,
                            need > 0 ? work.data_ptr() : nullptr, need);
        });
        return THPVariable_Wrap(dx);
    });
}

// linear_dw(dy, x): dy [M, N]^T @ x [M, K], both bf16
PyObject* host_linear_dw(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject* {
        const Tensor *dy = plain(a[0], at::kBFloat16), *x = plain(a[1], at::kBFloat16);
        if (!dy || !x || dy->dim() != 2 || x->dim() != 2 || x->device() != dy->device() ||
            dy->size(0) != x->size(0))
            Py_RETURN_NONE;
        const int64_t m = dy->size(0), n = dy->size(1), k = x->size(1);
        if (n % 16 != 0 || k % 16 != 0) Py_RETURN_NONE;
        const int64_t need = g_lib.dw_size(m, n, k);
        if (need < 0) fail("linear_dw");
        const void* st = current_stream(*dy);
        Tensor work, dw;
        call("linear_dw", [&] {
            if (need > 0) work = workspace(need, *dy);
            dw = empty({n, k}, at::kBFloat16, *dy);
            return g_lib.dw(st, dy->data_ptr(), x->data_ptr(), dw.data_ptr(), m, n, k,
                            need > 0 ? work.data_ptr() : nullptr, need);
        });
        return THPVariable_Wrap(dw);
    });
}

// column_sum(dy): the column sums of a bf16 [M, N]
PyObject* host_column_sum(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 1, [&]() -> PyObject* {
        const Tensor* dy = plain(a[0], at::kBFloat16);
        if (!dy || dy->dim() != 2 || dy->size(1) % 16 != 0) Py_RETURN_NONE;
        const int64_t m = dy->size(0), n = dy->size(1), need = g_lib.colsum_size(m, n);
        if (need < 0) fail("column_sum");
        const void* st = current_stream(*dy);
        Tensor work, out;
        call("column_sum", [&] {
            work = workspace(std::max<int64_t>(need, 16), *dy);
            out = empty({n}, at::kBFloat16, *dy);
            return g_lib.colsum(st, dy->data_ptr(), out.data_ptr(), m, n, work.data_ptr(), need);
        });
        return THPVariable_Wrap(out);
    });
}

// quantize(x): ops.quantize's (int8 [.., K], fp32 [..])
PyObject* host_quantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 1, [&]() -> PyObject* {
        const Tensor* x = plain(a[0], at::kBFloat16);
        if (!x || x->dim() < 1) Py_RETURN_NONE;
        const int64_t k = x->size(-1), m = x->numel() / k;
        const void* st = current_stream(*x);
        Tensor q, s;
        call("quantize", [&] {
            q = empty(x->sizes(), at::kChar, *x);
            s = empty(x->sizes().slice(0, x->dim() - 1), at::kFloat, *x);
            return g_lib.quantize(st, x->data_ptr(), static_cast<int8_t*>(q.data_ptr()),
                                  static_cast<float*>(s.data_ptr()), m, k);
        });
        return pair(q, s);
    });
}

// ------------------------------------------------- MXFP4 and mixture of experts
// the library's number of a floating element type, -1 for any other
int32_t type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: return -1;
    }
}
const at::ScalarType kTypes[3] = {at::kBFloat16, at::kHalf, at::kFloat};

// a plain tensor (see plain) of bf16, fp16 or fp32
const Tensor* floating(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    return t.defined() && type_of(t) >= 0 ? plain(o, t.scalar_type()) : nullptr;
}
const Tensor* on(const Tensor* t, const Tensor& like) {
    return t && t->device() == like.device() ? t : nullptr;
}
int64_t scale_width(int64_t k) { return (k + 511) / 512 * 16; }

// codes and scales that belong together
bool mx_pair(PyObject* c, PyObject* s, const Tensor*& codes, const Tensor*& scales) {
    codes = plain(c, at::kByte);
    scales = codes ? on(plain(s, at::kByte), *codes) : nullptr;
    if (!scales || codes->dim() < 1 || codes->dim() != scales->dim()) return false;
    const int64_t d = codes->dim() - 1, k = codes->size(d) * 2;
    return codes->sizes().slice(0, d) == scales->sizes().slice(0, d) && k % 32 == 0 &&
           scales->size(d) == scale_width(k);
}

// a moe.Routing (the caller has seen that it is one)
struct Routing {
    const Tensor *order, *position, *rows, *offsets;
};
bool routing_arg(PyObject* o, const Tensor& like, Routing& r) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
    r.order = on(plain(PyTuple_GET_ITEM(o, 0), at::kInt), like);
    r.position = on(plain(PyTuple_GET_ITEM(o, 1), at::kInt), like);
    r.rows = on(plain(PyTuple_GET_ITEM(o, 2), at::kInt), like);
    r.offsets = on(plain(PyTuple_GET_ITEM(o, 3), at::kInt), like);
    return r.order && r.position && r.rows && r.offsets && r.position->dim() == 2 &&
           r.position->numel() == r.order->numel() && r.rows->numel() == r.order->numel() &&
           r.offsets->numel() >= 2;
}
const int32_t* ints(const Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); }
int32_t* ints(Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
const uint8_t* bytes(const Tensor* t) { return static_cast<const uint8_t*>(t->data_ptr()); }

// mx_quantize(x): mxfp4.quantize
PyObject* host_mx_quantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 1, [&]() -> PyObject* {
        const Tensor* x = floating(a[0]);
        if (!x || x->dim() < 1 || x->size(-1) % 32 != 0) Py_RETURN_NONE;
        const int64_t k = x->size(-1), m = x->numel() / k;
        const void* st = current_stream(*x);
        Tensor c, s;
        call("mxfp4.quantize", [&] {
            c = empty(with_last(*x, k / 2), at::kByte, *x);
            s = empty(with_last(*x, scale_width(k)), at::kByte, *x);
            return g_lib.mx_quantize(st, x->data_ptr(), type_of(*x), k,
                                     static_cast<uint8_t*>(c.data_ptr()),
                                     static_cast<uint8_t*>(s.data_ptr()), m, k);
        });
        return pair(c, s);
    });
}

// mx_dequantize(codes, scales, type): mxfp4.dequantize
PyObject* host_mx_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 3, [&]() -> PyObject* {
        const Tensor *c, *s;
        const long type = PyLong_AsLong(a[2]);
        if (type == -1 && PyErr_Occurred()) throw python_error();
        if (type < 0 || type > 2 || !mx_pair(a[0], a[1], c, s)) Py_RETURN_NONE;
        const int64_t k = c->size(-1) * 2, m = c->numel() / (k / 2);
        const void* st = current_stream(*c);
        Tensor out;
        call("mxfp4.dequantize", [&] {
            out = empty(with_last(*c, k), kTypes[type], *c);
            return g_lib.mx_dequantize(st, bytes(c), bytes(s), out.data_ptr(), int32_t(type), m, k);
        });
        return THPVariable_Wrap(out);
    });
}

// ---------------------------------------------------- forward, on checked tensors
Tensor run_linear(const Tensor& x, const Tensor& c, const Tensor& s, const Tensor* b) {
    const int64_t n = c.size(0), k = c.size(1) * 2, m = x.numel() / k;
    const int64_t need = g_lib.mx_linear_size(m, n, k);
    if (need < 0) fail("mxfp4.linear");
    const void* st = current_stream(x);
    Tensor work, y;
    call("mxfp4.linear", [&] {
        if (need > 0) work = workspace(need, x);
        y = empty(with_last(x, n), x.scalar_type(), x);
        return g_lib.mx_linear(st, x.data_ptr(), type_of(x), k, bytes(&c), bytes(&s),
                               b ? b->data_ptr() : nullptr, b ? type_of(*b) : 0, y.data_ptr(), m,
                               n, k, need > 0 ? work.data_ptr() : nullptr, need);
    });
    return y;
}
// `rows`: the tokens that the sorted rows are read from, null for x sorted already
Tensor run_grouped(const Tensor& x, const Tensor& c, const Tensor& s, const Tensor* rows,
                   const Tensor& offsets, int64_t r) {
    const int64_t e = c.size(0), n = c.size(1), k = c.size(2) * 2, t = x.size(0);
    const int64_t need = g_lib.mx_grouped_size(r, t, e, n, k);
    if (need < 0) fail("mxfp4.grouped_linear");
    const void* st = current_stream(x);
    Tensor work, y;
    call("mxfp4.grouped_linear", [&] {
        if (need > 0) work = workspace(need, x);
        y = empty({r, n}, x.scalar_type(), x);
        return g_lib.mx_grouped(st, x.data_ptr(), type_of(x), k, rows ? ints(rows) : nullptr, t,
                                bytes(&c), bytes(&s), ints(&offsets), e, y.data_ptr(), r, n, k,
                                need > 0 ? work.data_ptr() : nullptr, need);
    });
    return y;
}
Tensor run_dispatch(const Tensor& x, const Tensor& position, const Tensor& offsets) {
    const int64_t t = x.size(0), d = x.size(1), top = position.size(1);
    const void* st = current_stream(x);
    Tensor out;
    call("moe.dispatch", [&] {
        out = empty({t * top, d}, x.scalar_type(), x);
        return g_lib.moe_dispatch(st, x.data_ptr(), type_of(x), d, ints(&position), ints(&offsets),
                                  out.data_ptr(), t, top, offsets.numel() - 1, d);
    });
    return out;
}
Tensor run_combine(const Tensor& z, const Tensor* w, const Tensor& position,
                   const Tensor& offsets, int32_t type) {
    const int64_t t = position.size(0), top = position.size(1), d = z.size(1);
    const void* st = current_stream(z);
    Tensor out;
    call("moe.combine", [&] {
        out = empty({t, d}, kTypes[type], z);
        return g_lib.moe_combine(st, z.data_ptr(), type_of(z), d, ints(&position), ints(&offsets),
                                 w ? static_cast<const float*>(w->data_ptr()) : nullptr,
                                 out.data_ptr(), type, t, top, offsets.numel() - 1, d);
    });
    return out;
}

// ------------------------------------------------------------------- gradients
// The backward passes as autograd nodes of C++: they run in the engine's thread without the
// GIL, which the current stream's accessor alone takes.  What they compute is what the
// Python functions' backward computes, by the same library calls.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// f() with the GIL, a Python error carried to where the engine reports it
template <class F>
auto with_gil(const F& f) {
    struct Gil {
        PyGILState_STATE s = PyGILState_Ensure();
        ~Gil() { PyGILState_Release(s); }
    } gil;
    try {
        return f();
    } catch (python_error& e) {
        e.persist();
        throw;
    }
}
const void* stream_of(const Tensor& t) {
    return with_gil([&] { return current_stream(t); });
}
void check(int rc, const char* what) {
    if (rc != 0) throw std::runtime_error(std::string(what) + ": " + g_lib.last_error());
}
// x [.., n] as rows with a stride, a sign that is a flag of the view applied
struct Rows {
    Tensor t;
    int64_t ld;
};
Rows rows_of(const Tensor& x) {
    Tensor t = x.resolve_neg().reshape({-1, x.size(-1)});
    const bool many = t.size(0) > 1;
    if (t.stride(1) != 1 || (many && t.stride(0) < t.size(1))) t = t.contiguous();
    return {t, t.size(0) > 1 ? t.stride(0) : t.size(1)};
}
bool on_default_stream(const Tensor& t) {
    return c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device()).id() == 0;
}
// whether the current stream is being captured (with the GIL)
bool capturing() {
    if (!g_capturing) return false;
    PyObject* r = PyObject_CallNoArgs(g_capturing);
    if (!r) throw python_error();
    const bool yes = r == Py_True;
    Py_DECREF(r);
    return yes;
}
void refuse_if_capturing() {
    PyObject* module = PyImport_ImportModule("xpu_kernels._capture");
    PyObject* r = module ? PyObject_CallMethod(module, "refuse_default_stream_leaf", nullptr) : nullptr;
    Py_XDECREF(module);
    if (!r) throw python_error();
    Py_DECREF(r);
}

// The gradient of a leaf ends in a node that lives as long as any graph of the leaf and
// belongs to the stream that was current when it was made.  A backward pass that is captured
// makes that stream wait for the capturing one; the default stream cannot, and that ends the
// process.  So a node here, before it gives its gradients to the engine in a capture, looks at
// all nodes that the pass takes them to, and refuses to go on if one is of the default stream.
void check_backward(const variable_list& in) {
    const Tensor* some = nullptr;
    for (const Tensor& g : in)
        if (g.defined()) some = &g;
    if (!some || !some->is_cuda() || on_default_stream(*some)) return;
    if (!with_gil([] { return capturing(); })) return;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
    if (!node) return;
    // (empty: the pass goes to all of them)
    const auto* pass = torch::autograd::get_current_graph_task_exec_info();
    std::vector<torch::autograd::Node*> left{node.get()};
    std::unordered_set<torch::autograd::Node*> seen{node.get()};
    while (!left.empty()) {
        torch::autograd::Node* from = left.back();
        left.pop_back();
        for (const auto& edge : from->next_edges()) {
            torch::autograd::Node* to = edge.function.get();
            if (!to || !seen.insert(to).second) continue;
            if (pass && !pass->empty()) {
                const auto it = pass->find(to);
                if (it == pass->end() || !it->second.should_execute()) continue;
            }
            const auto made = to->stream();
            if (made && made->id() == 0) return with_gil([] { refuse_if_capturing(); });
            left.push_back(to);
        }
    }
}

// the gradients that f() gives, which have no derivative themselves: an error where one is
// asked for
template <class F>
variable_list once(const variable_list& in, const F& f) {
    check_backward(in);
    variable_list grads;
    {
        at::NoGradGuard no_grad;
        grads = f();
    }
    bool wanted = false;
    for (const Tensor& g : in) wanted |= g.defined() && g.requires_grad();
    if (!wanted || !at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable",
        int64_t(grads.size()));
    return (*error)(std::move(grads));
}
Tensor grad_dx(const Rows& d, const Tensor& c, const Tensor& s, const Tensor* offsets,
               int32_t type) {
    const Tensor& dy = d.t;
    const int64_t n = c.size(-2), k = c.size(-1) * 2, e = offsets ? c.size(0) : 0, r = dy.size(0);
    const int64_t need = g_lib.mx_dx_size(dy.data_ptr(), type_of(dy), d.ld, type, r, e, n, k);
    if (need < 0) check(1, "mxfp4 dx");
    Tensor work, dx = empty({r, k}, kTypes[type], dy);
    if (need > 0) work = workspace(need, dy);
    check(g_lib.mx_dx(stream_of(dy), dy.data_ptr(), type_of(dy), d.ld, bytes(&c), bytes(&s),
                      offsets ? ints(offsets) : nullptr, e, dx.data_ptr(), type, r, n, k,
                      need > 0 ? work.data_ptr() : nullptr, need), "mxfp4 dx");
    return dx;
}
Tensor grad_sum(const Tensor& dxs, const Tensor& position, const Tensor& offsets, int32_t type) {
    const Rows z = rows_of(dxs);
    const int64_t t = position.size(0), top = position.size(1), d = z.t.size(1);
    Tensor out = empty({t, d}, kTypes[type], dxs);
    check(g_lib.moe_combine(stream_of(dxs), z.t.data_ptr(), type_of(dxs), z.ld, ints(&position),
                            ints(&offsets), nullptr, out.data_ptr(), type, t, top,
                            offsets.numel() - 1, d), "moe.combine");
    return out;
}
// dy's column sums in the bias's type
Tensor grad_bias(const Rows& dy, int32_t type) {
    const int64_t m = dy.t.size(0), n = dy.t.size(1), need = g_lib.mx_dbias_size(m, n);
    if (need < 0) check(1, "mxfp4 bias gradient");
    Tensor work = workspace(need, dy.t), out = empty({n}, kTypes[type], dy.t);
    check(g_lib.mx_dbias(stream_of(dy.t), dy.t.data_ptr(), type_of(dy.t), dy.ld, out.data_ptr(), type,
                         m, n, work.data_ptr(), need), "mxfp4 bias gradient");
    return out;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& c, const Tensor& s,
                          const std::optional<Tensor>& b) {
        ctx->save_for_backward({c, s});
        ctx->saved_data["bias"] = int64_t(b ? type_of(*b) : -1);
        return run_linear(x, c, s, b ? &*b : nullptr);
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &dy = in[0], &c = saved[0];
            const auto bias = int32_t(ctx->saved_data["bias"].toInt());
            const Rows rows = rows_of(dy);
            Tensor dx, db;
            if (ctx->needs_input_grad(0))
                dx = grad_dx(rows, c, saved[1], nullptr, type_of(dy)).reshape(with_last(dy, c.size(1) * 2));
            if (bias >= 0 && ctx->needs_input_grad(3)) db = grad_bias(rows, bias);
            return {dx, Tensor(), Tensor(), db};
        });
    }
};

struct GroupedFn : torch::autograd::Function<GroupedFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& c, const Tensor& s,
                          const Tensor& position, const Tensor& rows, const Tensor& offsets,
                          bool gather) {
        ctx->save_for_backward({c, s, position, offsets});
        ctx->saved_data["gather"] = gather;
        return run_grouped(x, c, s, gather ? &rows : nullptr, offsets, rows.numel());
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &dy = in[0], &offsets = saved[3];
            const bool gather = ctx->saved_data["gather"].toBool();
            // a token's rows are summed in fp32 and rounded once
            Tensor dx = grad_dx(rows_of(dy), saved[0], saved[1], &offsets, gather ? 2 : type_of(dy));
            if (gather) dx = grad_sum(dx, saved[2], offsets, type_of(dy));
            return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        });
    }
};

struct DispatchFn : torch::autograd::Function<DispatchFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position,
                          const Tensor& offsets) {
        ctx->save_for_backward({position, offsets});
        return run_dispatch(x, position, offsets);
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            return {grad_sum(in[0], saved[0], saved[1], type_of(in[0])), Tensor(), Tensor()};
        });
    }
};

struct CombineFn : torch::autograd::Function<CombineFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& w,
                          const Tensor& position, const Tensor& offsets) {
        ctx->save_for_backward({z, w, position, offsets});
        return run_combine(z, &w, position, offsets, type_of(z));
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &z = saved[0], &w = saved[1], &position = saved[2], &offsets = saved[3];
            const Rows dy = rows_of(in[0]);
            const int64_t t = position.size(0), top = position.size(1), d = z.size(1);
            Tensor dz = empty({t * top, d}, z.scalar_type(), z), dw = empty({t, top}, at::kFloat, z);
            check(g_lib.moe_combine_grad(stream_of(z), dy.t.data_ptr(), type_of(z), dy.ld, z.data_ptr(),
                                         d, ints(&position), ints(&offsets),
                                         static_cast<const float*>(w.data_ptr()), dz.data_ptr(),
                                         static_cast<float*>(dw.data_ptr()), t, top,
                                         offsets.numel() - 1, d), "moe.combine (gradient)");
            return {dz, dw, Tensor(), Tensor()};
        });
    }
};

// a forward-mode tangent, which the Python path refuses
bool has_tangent(const Tensor& a, const Tensor* b = nullptr) {
    return a._fw_grad(0).defined() || (b && b->_fw_grad(0).defined());
}
bool wants_grad(const Tensor& a, const Tensor* b = nullptr) {
    return at::GradMode::is_enabled() && (a.requires_grad() || (b && b->requires_grad()));
}

// -------------------------------------------------- functions of xpu_kernels.mxfp4, moe
// mx_linear(x, codes, scales, bias): mxfp4.linear
PyObject* host_mx_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 4, [&]() -> PyObject* {
        const Tensor* x = floating(a[0]);
        const Tensor *c, *s, *b = nullptr;
        if (!x || x->dim() < 1 || !mx_pair(a[1], a[2], c, s) || c->dim() != 2 || !on(c, *x) ||
            x->size(-1) != c->size(1) * 2)
            Py_RETURN_NONE;
        if (a[3] != Py_None) {
            b = on(floating(a[3]), *x);
            if (!b || b->dim() != 1 || b->numel() != c->size(0)) Py_RETURN_NONE;
        }
        if (has_tangent(*x, b)) Py_RETURN_NONE;
        if (!wants_grad(*x, b)) return THPVariable_Wrap(run_linear(*x, *c, *s, b));
        return THPVariable_Wrap(LinearFn::apply(*x, *c, *s, b ? std::optional<Tensor>(*b) : std::nullopt));
    });
}

// mx_grouped(x, codes, scales, routing, gather): mxfp4.grouped_linear
PyObject* host_mx_grouped(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 5, [&]() -> PyObject* {
        const Tensor* x = floating(a[0]);
        const Tensor *c, *s;
        Routing r;
        if (!x || x->dim() != 2 || !mx_pair(a[1], a[2], c, s) || c->dim() != 3 || !on(c, *x) ||
            !routing_arg(a[3], *x, r))
            Py_RETURN_NONE;
        const int gather = PyObject_IsTrue(a[4]);
        if (gather < 0) throw python_error();
        const int64_t rows = r.order->numel();
        if (x->size(1) != c->size(2) * 2 || r.offsets->numel() != c->size(0) + 1 ||
            x->size(0) != (gather ? r.position->size(0) : rows) || has_tangent(*x))
            Py_RETURN_NONE;
        if (!wants_grad(*x))
            return THPVariable_Wrap(run_grouped(*x, *c, *s, gather ? r.rows : nullptr, *r.offsets, rows));
        return THPVariable_Wrap(GroupedFn::apply(*x, *c, *s, *r.position, *r.rows, *r.offsets, gather != 0));
    });
}

// moe_sort(ids, n_experts): the four tensors of moe.sort's Routing
PyObject* host_moe_sort(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject* {
        const Tensor* ids = plain(a[0], at::kInt);
        const bool wide = !ids;
        if (wide) ids = plain(a[0], at::kLong);
        if (!ids || ids->dim() != 2 || !PyLong_CheckExact(a[1])) Py_RETURN_NONE;
        const long long e = PyLong_AsLongLong(a[1]);
        if (e == -1 && PyErr_Occurred()) throw python_error();
        if (e < 1 || e > 1024) Py_RETURN_NONE;
        const int64_t t = ids->size(0), top = ids->size(1);
        const int64_t need = g_lib.moe_sort_size(t, top, e);
        if (need < 0) fail("moe.sort");
        const void* st = current_stream(*ids);
        Tensor work, order, position, rows, offsets;
        call("moe.sort", [&] {
            if (need > 0) work = workspace(need, *ids);
            order = empty({t * top}, at::kInt, *ids);
            position = empty({t, top}, at::kInt, *ids);
            rows = empty({t * top}, at::kInt, *ids);
            offsets = empty({e + 1}, at::kInt, *ids);
            return g_lib.moe_sort(st, ids->data_ptr(), wide, ints(order), ints(position),
                                  ints(rows), ints(offsets), t, top, e,
                                  need > 0 ? work.data_ptr() : nullptr, need);
        });
        PyObject* out = PyTuple_New(4);
        if (!out) throw python_error();
        const Tensor all[4] = {order, position, rows, offsets};
        for (int i = 0; i < 4; ++i) {
            PyObject* o = THPVariable_Wrap(all[i]);
            if (!o) {
                Py_DECREF(out);
                throw python_error();
            }
            PyTuple_SET_ITEM(out, i, o);
        }
        return out;
    });
}

// moe_dispatch(x, routing): moe.dispatch
PyObject* host_moe_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject* {
        const Tensor* x = floating(a[0]);
        Routing r;
        if (!x || x->dim() != 2 || !routing_arg(a[1], *x, r) || x->size(0) != r.position->size(0) ||
            has_tangent(*x))
            Py_RETURN_NONE;
        if (!wants_grad(*x)) return THPVariable_Wrap(run_dispatch(*x, *r.position, *r.offsets));
        return THPVariable_Wrap(DispatchFn::apply(*x, *r.position, *r.offsets));
    });
}

// moe_combine(z, routing, weights): moe.combine, fp32 weights
PyObject* host_moe_combine(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 3, [&]() -> PyObject* {
        const Tensor* z = floating(a[0]);
        Routing r;
        if (!z || z->dim() != 2 || !routing_arg(a[1], *z, r)) Py_RETURN_NONE;
        const Tensor* w = on(plain(a[2], at::kFloat), *z);
        const int64_t t = r.position->size(0), top = r.position->size(1);
        if (!w || w->dim() != 2 || w->size(0) != t || w->size(1) != top || z->size(0) != t * top ||
            has_tangent(*z, w))
            Py_RETURN_NONE;
        if (!wants_grad(*z, w))
            return THPVariable_Wrap(run_combine(*z, w, *r.position, *r.offsets, type_of(*z)));
        return THPVariable_Wrap(CombineFn::apply(*z, *w, *r.position, *r.offsets));
    });
}

// ------------------------------------------------ xpu_kernels.norm, moe.route, rope
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
PyObject* wrapped(const variable_list& v) {
    PyObject* out = PyTuple_New(Py_ssize_t(v.size()));
    if (!out) throw python_error();
    for (size_t i = 0; i < v.size(); ++i) {
        PyObject* o = v[i].defined() ? THPVariable_Wrap(v[i]) : Py_NewRef(Py_None);
        if (!o) {
            Py_DECREF(out);
            throw python_error();
        }
        PyTuple_SET_ITEM(out, Py_ssize_t(i), o);
    }
    return out;
}
// an int or float object's value
bool number(PyObject* o, double& v) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
    v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool whole(PyObject* o, int64_t lo, int64_t hi, int64_t& v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over) return false;
    return v >= lo && v <= hi;
}
const std::optional<Tensor> maybe(const Tensor* t) { return t ? std::optional<Tensor>(*t) : std::nullopt; }

// The rows of a tensor as norm.py's _runs and _lines see them: runs of `inner` rows, ld apart,
// runs outer apart.
struct Lines {
    int64_t inner = 1, ld = 0, outer = 0;
};
bool runs_of(const Tensor& t, Lines& l) {
    const int64_t k = t.size(-1);
    if (t.stride(-1) != 1 && k > 1) return false;
    int64_t n[2] = {0, 0}, s[2] = {k, k};
    int levels = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (levels && t.stride(d) == n[levels - 1] * s[levels - 1]) {
            n[levels - 1] *= t.size(d);
        } else {
            if (levels == 2) return false;
            n[levels] = t.size(d);
            s[levels++] = t.stride(d);
        }
    }
    if (levels && s[0] < k) return false;
    l = levels == 2 ? Lines{n[0], s[0], s[1]} : Lines{1, s[0], s[0]};
    return true;
}
// the same in runs of `inner`
bool in_runs(Lines& l, int64_t inner) {
    if (l.inner == inner) return true;
    if (l.inner != 1) return false;
    l = Lines{inner, l.outer, l.outer * inner};
    return true;
}
// a plain tensor (see plain) of a floating type whose rows lie in runs, of any alignment
const Tensor* lines_arg(PyObject* o, Lines& l) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || type_of(t) < 0 ||
        t.key_set().has_any(kWrapped) || !t.has_storage() || t.dim() < 1 || t.numel() == 0 ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % t.element_size() != 0 || !runs_of(t, l))
        return nullptr;
    return &t;
}

// A forward call of a capture whose gradient would lead to a graph of the default stream (see
// check_backward), at once or through up to 16 views and other nodes of one input, is refused:
// most captured steps are stopped before their backward pass.  (Also where no backward pass
// follows: without gradient mode nothing is refused.)
void check_leaf(const Tensor* t) {
    if (!t || !t->requires_grad()) return;
    if (on_default_stream(*t)) return;
    std::shared_ptr<torch::autograd::Node> node = t->grad_fn();
    if (!node) node = torch::autograd::impl::try_get_grad_accumulator(*t);
    for (int far = 0; node && far < 16; ++far) {
        const auto made = node->stream();
        if (made && made->id() == 0) return refuse_if_capturing();
        std::shared_ptr<torch::autograd::Node> next;
        int inputs = 0;
        for (const auto& edge : node->next_edges())
            if (edge.is_valid() && inputs++ == 0) next = edge.function;
        node = inputs == 1 ? next : nullptr;
    }
}

// x, weight or None, eps, residual or None of a norm
struct NormCall {
    const Tensor *x = nullptr, *w = nullptr, *r = nullptr;
    Lines lx, lr;
    double eps = 0;
};
bool norm_call(PyObject* const* a, NormCall& c) {
    c.x = lines_arg(a[0], c.lx);
    if (!c.x || c.x->size(-1) > int64_t(1) << 24 || !number(a[2], c.eps) || !(c.eps >= 0)) return false;
    if (a[1] != Py_None) {
        c.w = on(floating(a[1]), *c.x);
        if (!c.w || c.w->dim() != 1 || c.w->numel() != c.x->size(-1)) return false;
    }
    if (a[3] != Py_None) {
        c.r = on(lines_arg(a[3], c.lr), *c.x);
        if (!c.r || c.r->scalar_type() != c.x->scalar_type() || c.r->sizes() != c.x->sizes()) return false;
        const int64_t inner = std::max(c.lx.inner, c.lr.inner);
        if (!in_runs(c.lx, inner) || !in_runs(c.lr, inner)) return false;
    }
    return !has_tangent(*c.x, c.w) && !(c.r && has_tangent(*c.r));
}

// (y, h or undefined)
std::array<Tensor, 2> run_norm(const Tensor& x, const Lines& lx, const Tensor* w, double eps,
                               const Tensor* r, const Lines& lr) {
    const int64_t k = x.size(-1), m = x.numel() / k;
    const void* st = current_stream(x);
    Tensor y, h;
    call("norm.rms_norm", [&] {
        const c10::DeviceGuard on_x(x.device());
        y = empty(x.sizes(), x.scalar_type(), x);
        if (r) h = empty(x.sizes(), x.scalar_type(), x);
        return g_lib.rms_norm(st, x.data_ptr(), type_of(x), lx.ld, lx.outer, r ? r->data_ptr() : nullptr,
                              lr.ld, lr.outer, lx.inner, w ? w->data_ptr() : nullptr, w ? type_of(*w) : 0, float(eps), ptr(h),
                              y.data_ptr(), m, k);
    });
    return {y, h};
}

struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w,
                                 double eps, const std::optional<Tensor>& r, const Lines& lx,
                                 const Lines& lr) {
        ctx->set_materialize_grads(false);
        auto [y, h] = run_norm(x, lx, w ? &*w : nullptr, eps, r ? &*r : nullptr, lr);
        ctx->save_for_backward({r ? h : x, w ? *w : Tensor()});
        ctx->saved_data["eps"] = eps;
        if (r) return {y, h};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &h = saved[0], &w = saved[1], &dy = in[0];
            const Tensor dh = in.size() > 1 ? in[1] : Tensor();
            const double eps = ctx->saved_data["eps"].toDouble();
            const bool want = w.defined() && ctx->needs_input_grad(1);
            Tensor dx, dw;
            if (!dy.defined()) {
                dx = dh;
                if (want) dw = at::zeros_like(w);
            } else {
                const c10::DeviceGuard on_h(h.device());
                const int64_t k = h.size(-1), m = h.numel() / k;
                // h as it was normalised, its gradients in the same runs or copied
                Lines lh, lg, lb;
                if (!runs_of(h, lh)) check(1, "norm.rms_norm (gradient)");
                auto lines = [&](const Tensor& t, Lines& l) {
                    const Tensor r = t.resolve_neg();
                    if (runs_of(r, l) && in_runs(l, lh.inner)) return r;
                    l = Lines{1, k, k};
                    in_runs(l, lh.inner);
                    return r.contiguous();
                };
                const Tensor g = lines(dy, lg);
                Tensor b;
                if (dh.defined()) b = lines(dh, lb);
                const int64_t need = want ? g_lib.rms_norm_grad_size(m, k) : 0;
                if (need < 0) check(1, "norm.rms_norm (gradient)");
                Tensor work;
                if (want) {
                    work = workspace(need, h);
                    dw = empty({k}, w.scalar_type(), h);
                }
                dx = empty(h.sizes(), h.scalar_type(), h);
                check(g_lib.rms_norm_grad(stream_of(h), g.data_ptr(), type_of(h), lg.ld, lg.outer,
                                          h.data_ptr(), lh.ld, lh.outer, ptr(w),
                                          w.defined() ? type_of(w) : 0, ptr(b), lb.ld, lb.outer, lh.inner,
                                          float(eps), dx.data_ptr(), ptr(dw), m, k, ptr(work), need),
                      "norm.rms_norm (gradient)");
            }
            // x, weight, eps, residual, their rows (needs_input_grad counts the tensors that are there)
            const bool to_r = in.size() > 1 && ctx->needs_input_grad(w.defined() ? 2 : 1);
            return {ctx->needs_input_grad(0) ? dx : Tensor(), dw, Tensor(), to_r ? dx : Tensor(), Tensor(),
                    Tensor()};
        });
    }
};

// rms_norm(x, weight, eps, residual): norm.rms_norm
PyObject* host_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 4, [&]() -> PyObject* {
        NormCall c;
        if (!norm_call(a, c)) Py_RETURN_NONE;
        if (wants_grad(*c.x, c.w) || (c.r && wants_grad(*c.r))) {
            for (const Tensor* t : {c.x, c.w, c.r}) check_leaf(t);
            const variable_list out = NormFn::apply(*c.x, maybe(c.w), c.eps, maybe(c.r), c.lx, c.lr);
            return c.r ? wrapped(out) : THPVariable_Wrap(out[0]);
        }
        auto [y, h] = run_norm(*c.x, c.lx, c.w, c.eps, c.r, c.lr);
        return c.r ? pair(y, h) : THPVariable_Wrap(y);
    });
}

// rms_norm_int8(x, weight, eps, residual, rotate): norm.rms_norm_int8 of inputs without gradients
PyObject* host_rms_norm_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 5, [&]() -> PyObject* {
        NormCall c;
        if (!norm_call(a, c) || wants_grad(*c.x, c.w) || (c.r && wants_grad(*c.r))) Py_RETURN_NONE;
        const int rotate = PyObject_IsTrue(a[4]);
        if (rotate < 0) throw python_error();
        const Tensor& x = *c.x;
        const int64_t k = x.size(-1), m = x.numel() / k;
        if (rotate && k % 256 != 0) Py_RETURN_NONE;
        const void* st = current_stream(x);
        Tensor q, s, h;
        call("norm.rms_norm_int8", [&] {
            const c10::DeviceGuard on_x(x.device());
            q = empty(x.sizes(), at::kChar, x);
            s = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
            if (c.r) h = empty(x.sizes(), x.scalar_type(), x);
            return g_lib.rms_norm_int8(st, x.data_ptr(), type_of(x), c.lx.ld, c.lx.outer,
                                       c.r ? c.r->data_ptr() : nullptr, c.lr.ld, c.lr.outer, c.lx.inner,
                                       c.w ? c.w->data_ptr() : nullptr, c.w ? type_of(*c.w) : 0,
                                       float(c.eps), ptr(h), static_cast<int8_t*>(q.data_ptr()),
                                       static_cast<float*>(s.data_ptr()), rotate, m, k);
        });
        return c.r ? wrapped({q, s, h}) : pair(q, s);
    });
}

struct RouteHow {
    int32_t sigmoid, renormalize;
    int64_t groups, top_groups;
    double scale;
};
std::array<Tensor, 2> run_route(const Tensor& l, const Tensor* b, const RouteHow& how, int64_t top) {
    const int64_t t = l.size(0), e = l.size(1);
    const void* st = current_stream(l);
    Tensor ids, w;
    call("moe.route", [&] {
        const c10::DeviceGuard on_l(l.device());
        ids = empty({t, top}, at::kInt, l);
        w = empty({t, top}, at::kFloat, l);
        return g_lib.moe_route(st, l.data_ptr(), type_of(l), e,
                               b ? static_cast<const float*>(b->data_ptr()) : nullptr, how.sigmoid,
                               how.groups, how.top_groups, how.renormalize, float(how.scale),
                               ints(ids), static_cast<float*>(w.data_ptr()), t, e, top);
    });
    return {ids, w};
}

struct RouteFn : torch::autograd::Function<RouteFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& l, const std::optional<Tensor>& b,
                                 int64_t sigmoid, int64_t renormalize, int64_t groups,
                                 int64_t top_groups, double scale, int64_t top) {
        ctx->set_materialize_grads(false);
        const RouteHow how{int32_t(sigmoid), int32_t(renormalize), groups, top_groups, scale};
        auto [ids, w] = run_route(l, b ? &*b : nullptr, how, top);
        ctx->save_for_backward({l, ids});
        ctx->saved_data["sigmoid"] = sigmoid;
        ctx->saved_data["renormalize"] = renormalize;
        ctx->saved_data["scale"] = scale;
        ctx->mark_non_differentiable({ids});
        return {ids, w};
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            variable_list out(8);
            if (!in[1].defined()) return out;
            const variable_list saved = ctx->get_saved_variables();
            const Tensor &l = saved[0], &ids = saved[1];
            const c10::DeviceGuard on_l(l.device());
            const Tensor dw = in[1].resolve_neg().contiguous();
            const int64_t t = l.size(0), e = l.size(1);
            out[0] = empty({t, e}, l.scalar_type(), l);
            check(g_lib.moe_route_grad(stream_of(l), l.data_ptr(), type_of(l), e, ints(&ids),
                                       static_cast<const float*>(dw.data_ptr()),
                                       int32_t(ctx->saved_data["sigmoid"].toInt()),
                                       int32_t(ctx->saved_data["renormalize"].toInt()),
                                       float(ctx->saved_data["scale"].toDouble()), out[0].data_ptr(),
                                       t, e, ids.size(1)), "moe.route (gradient)");
            return out;
        });
    }
};

// moe_route(logits, top, scores, bias, groups, top_groups, renormalize, scale): moe.route
PyObject* host_moe_route(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 8, [&]() -> PyObject* {
        const Tensor* l = floating(a[0]);
        const Tensor* b = nullptr;
        if (!l || l->dim() != 2 || l->size(1) > 1024 || has_tangent(*l) || !PyUnicode_CheckExact(a[2]))
            Py_RETURN_NONE;
        RouteHow how;
        const int64_t e = l->size(1);
        int64_t top;
        how.sigmoid = PyUnicode_CompareWithASCIIString(a[2], "sigmoid") == 0;
        if (!how.sigmoid && PyUnicode_CompareWithASCIIString(a[2], "softmax") != 0) Py_RETURN_NONE;
        if (a[3] != Py_None) {
            b = on(plain(a[3], at::kFloat), *l);
            if (!b || b->dim() != 1 || b->numel() != e || has_tangent(*b) || wants_grad(*b)) Py_RETURN_NONE;
        }
        if (!whole(a[1], 1, e < 64 ? e : 64, top) || !whole(a[4], 1, 64, how.groups) ||
            !whole(a[5], 1, how.groups, how.top_groups) || e % how.groups != 0 ||
            top > how.top_groups * (e / how.groups) || !number(a[7], how.scale))
            Py_RETURN_NONE;
        const int renormalize = PyObject_IsTrue(a[6]);
        if (renormalize < 0) throw python_error();
        how.renormalize = renormalize;
        if (wants_grad(*l)) {
            check_leaf(l);
            return wrapped(RouteFn::apply(*l, maybe(b), int64_t(how.sigmoid), int64_t(how.renormalize),
                                          how.groups, how.top_groups, how.scale, top));
        }
        auto [ids, w] = run_route(*l, b, how, top);
        return pair(ids, w);
    });
}

// A tensor of heads [B, S, H, D] of any strides but a contiguous head dimension; otherwise
// as plain, aligned to its elements
const Tensor* heads_arg(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || type_of(t) < 0 ||
        t.key_set().has_any(kWrapped) || !t.has_storage() || t.dim() != 4 || t.numel() == 0 ||
        t.stride(3) != 1 || t.size(3) > 4096 ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % t.element_size() != 0)
        return nullptr;
    return &t;
}
const Tensor* positions_arg(PyObject* o, const Tensor& q) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || t.device() != q.device() ||
        t.key_set().has_any(kWrapped) || !t.has_storage() || t.numel() == 0 || wants_grad(t))
        return nullptr;
    const auto type = t.scalar_type();
    if (type != at::kInt && type != at::kLong && type != at::kFloat) return nullptr;
    const bool fits = t.dim() == 3 ? t.size(1) == q.size(0) && t.size(2) == q.size(1)
                                   : t.dim() == 2 && t.size(1) == q.size(1);
    return fits && t.size(0) >= 1 && t.size(0) <= 16 ? &t : nullptr;
}
// an empty result in x's layout where that is dense (rope._like)
Tensor like_heads(const Tensor& x) {
    Tensor out = at::empty_like(x);
    return out.stride(3) == 1 ? out : empty(x.sizes(), x.scalar_type(), x);
}
struct Strides {
    int64_t s[6];
    Strides(const Tensor& x, const Tensor& out)
        : s{x.stride(0), x.stride(1), x.stride(2), out.stride(0), out.stride(1), out.stride(2)} {}
};
// q and, where it is defined, k (of contiguous heads) into oq and ok
int turn(const void* st, const Tensor& q, const Tensor& k, const Tensor& positions,
         const Tensor& inv_freq, const Tensor& axis, bool inverse, bool split, Tensor& oq, Tensor& ok) {
    const c10::DeviceGuard on_q(q.device());
    oq = like_heads(q);
    if (k.defined()) ok = like_heads(k);
    const Strides qs(q, oq), ks(k.defined() ? k : q, k.defined() ? ok : oq);
    const int d = int(positions.dim());
    const int64_t ps[3] = {positions.stride(0), d == 2 ? 0 : positions.stride(1), positions.stride(d - 1)};
    const auto type = positions.scalar_type();
    return g_lib.rope_axes(st, q.data_ptr(), oq.data_ptr(), qs.s, q.size(2), ptr(k), ptr(ok),
                           k.defined() ? ks.s : nullptr, k.defined() ? k.size(2) : 0, type_of(q),
                           positions.data_ptr(), type == at::kInt ? 0 : type == at::kLong ? 1 : 2, ps,
                           positions.size(0), static_cast<const double*>(inv_freq.data_ptr()),
                           ints(&axis), axis.numel(), inverse, split, q.size(0), q.size(1), q.size(3));
}

struct TurnFn : torch::autograd::Function<TurnFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k,
                                 const Tensor& positions, const Tensor& inv_freq, const Tensor& axis,
                                 bool split) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, inv_freq, axis});
        ctx->saved_data["split"] = split;
        const void* st = current_stream(q);
        Tensor oq, ok;
        call("rope.rotate_axes", [&] {
            return turn(st, q, k ? *k : Tensor(), positions, inv_freq, axis, false, split, oq, ok);
        });
        if (k) return {oq, ok};
        return {oq};
    }
    static variable_list backward(AutogradContext* ctx, variable_list in) {
        return once(in, [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const bool split = ctx->saved_data["split"].toBool();
            // gradients of any strides, a sign that is a flag of the view applied
            auto heads = [](const Tensor& t) {
                const Tensor r = t.resolve_neg();
                return r.stride(3) == 1 || r.size(3) == 1 ? r : r.contiguous();
            };
            Tensor dq, dk, oq, ok;
            if (in[0].defined() && ctx->needs_input_grad(0)) dq = heads(in[0]);
            if (in.size() > 1 && in[1].defined() && ctx->needs_input_grad(1)) dk = heads(in[1]);
            if (dq.defined()) {
                check(turn(stream_of(dq), dq, dk, saved[0], saved[1], saved[2], true, split, oq, ok),
                      "rope.rotate_axes");
            } else if (dk.defined()) {
                check(turn(stream_of(dk), dk, Tensor(), saved[0], saved[1], saved[2], true, split, ok, oq),
                      "rope.rotate_axes");
            }
            return {oq, ok, Tensor(), Tensor(), Tensor(), Tensor()};
        });
    }
};

// rotate_axes(q, k, positions, frequencies, split_half): rope.rotate_axes (the caller has
// seen that frequencies is an AxisFrequencies)
PyObject* host_rotate_axes(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, 5, [&]() -> PyObject* {
        const Tensor *q = heads_arg(a[0]), *k = nullptr;
        if (!q || !PyTuple_Check(a[3]) || PyTuple_GET_SIZE(a[3]) != 2) Py_RETURN_NONE;
        if (a[1] != Py_None) {
            k = on(heads_arg(a[1]), *q);
            if (!k || k->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) ||
                k->size(1) != q->size(1) || k->size(3) != q->size(3))
                Py_RETURN_NONE;
        }
        const Tensor* positions = positions_arg(a[2], *q);
        const Tensor* inv_freq = on(plain(PyTuple_GET_ITEM(a[3], 0), at::kDouble), *q);
        const Tensor* axis = on(plain(PyTuple_GET_ITEM(a[3], 1), at::kInt), *q);
        if (!positions || !inv_freq || !axis || inv_freq->dim() != 1 || axis->dim() != 1 ||
            axis->numel() != inv_freq->numel() || axis->numel() > 512 || 2 * axis->numel() > q->size(3) ||
            q->size(2) + (k ? k->size(2) : 0) > 65536 || has_tangent(*q, k) || has_tangent(*positions) ||
            has_tangent(*inv_freq) || wants_grad(*inv_freq))
            Py_RETURN_NONE;
        const int split = PyObject_IsTrue(a[4]);
        if (split < 0) throw python_error();
        variable_list out(2);
        if (wants_grad(*q, k)) {
            check_leaf(q);
            check_leaf(k);
            const variable_list r = TurnFn::apply(*q, maybe(k), *positions, *inv_freq, *axis, split != 0);
            out[0] = r[0];
            if (k) out[1] = r[1];
        } else {
            const void* st = current_stream(*q);
            call("rope.rotate_axes", [&] {
                return turn(st, *q, k ? *k : Tensor(), *positions, *inv_freq, *axis, false, split != 0,
                            out[0], out[1]);
            });
        }
        return wrapped(out);
    });
}

// check_backward(gradients or Nones ..): for nodes of Python
PyObject* host_check_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, n_args, [&]() -> PyObject* {
        variable_list in;
        for (Py_ssize_t i = 0; i < n_args; ++i)
            if (THPVariable_Check(a[i])) in.push_back(THPVariable_Unpack(a[i]));
        check_backward(in);
        Py_RETURN_NONE;
    });
}

// check_leaves(tensors or Nones ..): check_leaf for calls that go through Python
PyObject* host_check_leaves(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded(n_args, n_args, [&]() -> PyObject* {
        for (Py_ssize_t i = 0; i < n_args; ++i)
            if (THPVariable_Check(a[i])) check_leaf(&THPVariable_Unpack(a[i]));
        Py_RETURN_NONE;
    });
}

// bind(addresses, raw_stream, packed): the library's entry points in Library's
// order, the current-stream accessor and the packed-weight registry
PyObject* host_bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 3 || !PyTuple_CheckExact(a[0]) || PyTuple_GET_SIZE(a[0]) != kEntries ||
        !PyCallable_Check(a[1]) || !PyDict_CheckExact(a[2])) {
        PyErr_SetString(PyExc_TypeError, "bind(tuple of addresses, callable, dict)");
        return nullptr;
    }
    std::array<void*, kEntries> p;
    for (int i = 0; i < kEntries; ++i) {
        p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
        if (!p[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
            return nullptr;
        }
    }
    std::memcpy(static_cast<void*>(&g_lib), p.data(), sizeof(g_lib));
    Py_XSETREF(g_raw_stream, Py_NewRef(a[1]));
    Py_XSETREF(g_packed, Py_NewRef(a[2]));
    PyObject* torch_c = PyImport_ImportModule("torch._C");
    PyObject* asks = torch_c ? PyObject_GetAttrString(torch_c, "_cuda_isCurrentStreamCapturing") : nullptr;
    Py_XDECREF(torch_c);
    if (!asks) PyErr_Clear();                        // (torch without a device: nothing is captured)
    Py_XSETREF(g_capturing, asks);
    Py_RETURN_NONE;
}

#define XPU_HOST(name, fn) \
    {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fn)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {XPU_HOST("bind", host_bind),
                          XPU_HOST("linear", host_linear),
                          XPU_HOST("linear_acc", host_linear_acc),
                          XPU_HOST("ffn", host_ffn),
                          XPU_HOST("backward", host_backward),
                          XPU_HOST("linear_dx", host_linear_dx),
                          XPU_HOST("linear_dw", host_linear_dw),
                          XPU_HOST("column_sum", host_column_sum),
                          XPU_HOST("quantize", host_quantize),
                          XPU_HOST("mx_quantize", host_mx_quantize),
                          XPU_HOST("mx_dequantize", host_mx_dequantize),
                          XPU_HOST("mx_linear", host_mx_linear),
                          XPU_HOST("mx_grouped", host_mx_grouped),
                          XPU_HOST("moe_sort", host_moe_sort),
                          XPU_HOST("moe_dispatch", host_moe_dispatch),
                          XPU_HOST("moe_combine", host_moe_combine),
                          XPU_HOST("rms_norm", host_rms_norm),
                          XPU_HOST("rms_norm_int8", host_rms_norm_int8),
                          XPU_HOST("moe_route", host_moe_route),
                          XPU_HOST("rotate_axes", host_rotate_axes),
                          XPU_HOST("check_leaves", host_check_leaves),
                          XPU_HOST("check_backward", host_check_backward),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host",
                       "The int8 API's hot calls in native code (see host_ops.cpp).", -1, kMethods};

// Tensors are read by the layout that torch's headers gave at build time, and
// another build of torch can export the same symbols over another layout: the
// module loads only into the Python and the torch (version and commit) that the
// Makefile found, XPU_BUILT_FOR = "3.10/2.10.0+rocm7.0/<commit>", and raises
// ImportError elsewhere.
bool built_for_this() {
    int major = 0, minor = 0;
    std::sscanf(Py_GetVersion(), "%d.%d", &major, &minor);
    PyObject* v = PyImport_ImportModule("torch.version");
    PyObject* version = v ? PyObject_GetAttrString(v, "__version__") : nullptr;
    PyObject* commit = version ? PyObject_GetAttrString(v, "git_version") : nullptr;
    PyObject* now = commit ? PyUnicode_FromFormat("%d.%d/%S/%S", major, minor, version, commit)
                           : nullptr;
    const bool ok = now && PyUnicode_CompareWithASCIIString(now, XPU_BUILT_FOR) == 0;
    if (!ok) {
        PyErr_Clear();
        PyErr_Format(PyExc_ImportError, "_host.so was built for " XPU_BUILT_FOR ", not %S",
                     now ? now : Py_None);
    }
    Py_XDECREF(now);
    Py_XDECREF(commit);
    Py_XDECREF(version);
    Py_XDECREF(v);
    return ok;
}

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    if (!built_for_this()) return nullptr;
    return PyModule_Create(&kModule);
}
