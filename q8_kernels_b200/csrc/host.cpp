// Host side of the ops in native code: argument checks, output allocation and the launch of one op per call from
// Python, as a CPython extension over the C ABI (fastcall, no binding layer).
//
// Every function here is the common case of the function of the same name in native.py and returns None for anything
// else: tensors that are not plain, dense CUDA tensors of the current device, active dispatch modes or transforms,
// shapes, types and alignments it does not know, and everything that is to be refused.  The Python function then does
// the whole of its own work, so what is accepted, what is refused and how is decided in one place.  An error of a
// launch itself is raised from here, by _lib.check.
//
// What it is for: a ctypes call with its argument conversions, torch.empty and the checks in Python cost 4 to 8 us an op,
// more than the kernels of a short call take.

#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/q8_kernels_b200.h"

namespace {

PyObject* g_check = nullptr;                                   // _lib.check(rc, op): raises Q8KernelError
constexpr int kMaxDevices = 64;
at::Tensor* g_status[kMaxDevices] = {};                        // the devices' status words (set_status_word)

using Dt = at::ScalarType;

int dt_code(Dt t) {
    switch (t) {
        case Dt::Float: return Q8K_DT_F32;
        case Dt::BFloat16: return Q8K_DT_BF16;
        case Dt::Float8_e4m3fn: return Q8K_DT_E4M3;
        case Dt::Char: return Q8K_DT_I8;
        default: return -1;                                    // not on a fast path
    }
}

// The arguments of one call.  `ok` turns false as soon as one of them is not what the fast path takes, their number first of
// all; from then on none is looked at any more.
struct Call {
    PyObject* const* args;
    bool ok;
    c10::DeviceIndex dev = -1;

    Call(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : args(a), ok(n == want) {
        // a transform, a tracer or a mode that wants to see the ops
        if (c10::impl::TorchDispatchModeTLS::any_modes_set()) ok = false;
        const auto tls = c10::impl::tls_local_dispatch_key_set();
        if (tls.included_.has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                                       c10::DispatchKey::FuncTorchDynamicLayerBackMode,
                                                       c10::DispatchKey::FuncTorchBatched,
                                                       c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::VmapMode,
                                                       c10::DispatchKey::Functionalize, c10::DispatchKey::Tracer,
                                                       c10::DispatchKey::Python, c10::DispatchKey::PreDispatch})))
            ok = false;
    }
    // A plain CUDA tensor of the device that is current; contiguous unless `strided`.
    const at::Tensor* tensor(int i, bool strided = false) { return ok ? tensor_of(args[i], strided) : nullptr; }
    const at::Tensor* tensor_of(PyObject* o, bool strided = false) {
        static const uint64_t plain =
            c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradCUDA,
                                 c10::DispatchKey::AutocastCUDA}).raw_repr();
        ok = false;
        if (!THPVariable_Check(o)) return nullptr;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || !t.is_cuda() || (t.key_set().raw_repr() & ~plain) != 0) return nullptr;
        if (!strided && !t.is_contiguous()) return nullptr;
        const c10::DeviceIndex d = t.device().index();
        if (dev < 0) {
            if (d >= kMaxDevices || d != c10::cuda::current_device()) return nullptr;
            dev = d;
        } else if (d != dev) {
            return nullptr;
        }
        ok = true;
        return &t;
    }
    const at::Tensor* tensor(int i, Dt type, bool strided = false) {
        const at::Tensor* t = tensor(i, strided);
        if (t != nullptr && t->scalar_type() != type) ok = false;
        return t;
    }
    const at::Tensor* optional(int i, Dt type) { return !ok || args[i] == Py_None ? nullptr : tensor(i, type); }
    Dt dtype(int i, Dt none) {
        if (!ok || args[i] == Py_None) return none;
        if (!THPDtype_Check(args[i])) { ok = false; return none; }
        return reinterpret_cast<THPDtype*>(args[i])->scalar_type;
    }
    bool flag(int i) {
        if (!ok) return false;
        if (args[i] == Py_True) return true;
        if (args[i] != Py_False) ok = false;
        return false;
    }
    long integer(int i) {
        if (!ok) return 0;
        if (!PyLong_CheckExact(args[i])) { ok = false; return 0; }
        const long v = PyLong_AsLong(args[i]);
        if (v < 0 || v > 0x7fffffff) { PyErr_Clear(); ok = false; }
        return v;
    }
    float real(int i) {
        if (!ok) return 0.f;
        if (!PyFloat_CheckExact(args[i])) { ok = false; return 0.f; }
        return (float)PyFloat_AS_DOUBLE(args[i]);
    }
    int* status() {
        if (ok && g_status[dev] == nullptr) ok = false;        // the Python path makes it
        return ok ? g_status[dev]->data_ptr<int>() : nullptr;
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
    void need(bool cond) { ok = ok && cond; }
    at::Tensor empty(at::IntArrayRef shape, Dt type) const {
        return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, dev)));
    }
};

// Allocation and launch without the interpreter lock, as torch and ctypes do them.  (The caller's references keep the
// arguments alive.)
struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <typename F> int launch(F&& f) {
    WithoutGil unlocked;
    return f();
}

// True when the launch was taken; otherwise the Python error is set.
bool launched(int rc, const char* op) {
    if (rc == Q8K_OK) return true;
    PyObject* r = PyObject_CallFunction(g_check, "is", rc, op);
    Py_XDECREF(r);
    if (r != nullptr) PyErr_SetString(PyExc_RuntimeError, "q8_kernels_b200: a launch failed");
    return false;
}

PyObject* wrap(at::Tensor&& t) { return THPVariable_Wrap(std::move(t)); }
PyObject* list2(at::Tensor&& a, at::Tensor&& b) {
    PyObject* l = PyList_New(2);
    if (l == nullptr) return nullptr;
    PyList_SET_ITEM(l, 0, wrap(std::move(a)));
    PyList_SET_ITEM(l, 1, wrap(std::move(b)));
    return l;
}
PyObject* tuple_of(at::Tensor (&t)[3]) {                       // of those that are defined
    PyObject* r = PyTuple_New(t[0].defined() + t[1].defined() + t[2].defined());
    if (r == nullptr) return nullptr;
    Py_ssize_t k = 0;
    for (at::Tensor& x : t)
        if (x.defined()) PyTuple_SET_ITEM(r, k++, wrap(std::move(x)));
    return r;
}

const void* cptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->const_data_ptr(); }
const float* fptr(const at::Tensor* t) { return static_cast<const float*>(cptr(t)); }
bool int_sized(int64_t v) { return v >= 0 && v <= 0x7fffffffLL; }
at::IntArrayRef lead(const at::Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }   // shape without the last dim
bool has_rows(const at::Tensor* t) { return t->dim() >= 1 && t->size(-1) > 0 && int_sized(t->size(-1)); }
bool quant_type(Dt t) { return t == Dt::Char || t == Dt::Float8_e4m3fn; }

#define FAST_BEGIN HANDLE_TH_ERRORS
#define FAST_END END_HANDLE_TH_ERRORS                          // torch's own exceptions, out of memory among them
#define OR_NONE(c) \
    if (!(c).ok) Py_RETURN_NONE

// ---------------------------------------------------------------- rows
// tokenwise_quant(x, out_type)
PyObject* tokenwise_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 2);
    const at::Tensor* x = c.tensor(0);
    const Dt out = c.dtype(1, Dt::Char);
    OR_NONE(c);
    c.need(has_rows(x) && quant_type(out) && dt_code(x->scalar_type()) >= 0);
    OR_NONE(c);
    const int dim = (int)x->size(-1);
    at::Tensor q, s;
    const int rc = launch([&] {
        q = c.empty(x->sizes(), out);
        s = c.empty(lead(*x), Dt::Float);
        return q8k_tokenwise_quant(cptr(x), dt_code(x->scalar_type()), q.data_ptr(), dt_code(out), s.data_ptr<float>(),
                                   x->numel() / dim, dim, dim, c.stream());
    });
    return launched(rc, "tokenwise_quant") ? list2(std::move(q), std::move(s)) : nullptr;
    FAST_END
}

// hadamard_quant(x, scale, out_type)
PyObject* hadamard_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 3);
    const at::Tensor* x = c.tensor(0);
    const float scale = c.real(1);
    const Dt out = c.dtype(2, Dt::Char);
    OR_NONE(c);
    c.need(has_rows(x) && quant_type(out) && dt_code(x->scalar_type()) >= 0);
    OR_NONE(c);
    const int dim = (int)x->size(-1);
    at::Tensor q, s;
    const int rc = launch([&] {
        q = c.empty(x->sizes(), out);
        s = c.empty(lead(*x), Dt::Float);
        return q8k_hadamard_quant(cptr(x), dt_code(x->scalar_type()), q.data_ptr(), dt_code(out), s.data_ptr<float>(),
                                  x->numel() / dim, dim, dim, scale, c.stream());
    });
    return launched(rc, "hadamard_quant") ? list2(std::move(q), std::move(s)) : nullptr;
    FAST_END
}

// fast_hadamard_transform(x, scale, out_type)
PyObject* fast_hadamard_transform(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 3);
    const at::Tensor* x = c.tensor(0);
    const float scale = c.real(1);
    OR_NONE(c);
    const Dt in = x->scalar_type();
    const Dt out = c.dtype(2, in);
    c.need(has_rows(x) && x->size(-1) % 8 == 0 && (in == Dt::BFloat16 || in == Dt::Float8_e4m3fn) && dt_code(out) >= 0);
    OR_NONE(c);
    const int dim = (int)x->size(-1);
    at::Tensor y;
    const int rc = launch([&] {
        y = c.empty(x->sizes(), out);
        return q8k_fast_hadamard_transform(cptr(x), dt_code(in), y.data_ptr(), dt_code(out), x->numel() / dim, dim, dim,
                                           scale, c.stream());
    });
    return launched(rc, "fast_hadamard_transform") ? wrap(std::move(y)) : nullptr;
    FAST_END
}

// norm_modulate_quant(x, mod_scale, mod_shift, out_type)
PyObject* norm_modulate_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 4);
    const at::Tensor* x = c.tensor(0, Dt::BFloat16);
    const at::Tensor* sc = c.tensor(1, Dt::BFloat16);
    const at::Tensor* sh = c.tensor(2, Dt::BFloat16);
    const Dt out = c.dtype(3, Dt::Char);
    OR_NONE(c);
    c.need(x->dim() == 3 && has_rows(x) && quant_type(out));
    OR_NONE(c);
    const int64_t B = x->size(0), S = x->size(1), dim = x->size(2);
    for (const at::Tensor* m : {sc, sh}) c.need(m->dim() == 3 && m->size(0) == B && m->size(1) == 1 && m->size(2) == dim);
    OR_NONE(c);
    at::Tensor q, s;
    const float scale = (float)(1.0 / std::sqrt((double)dim));
    const int rc = launch([&] {
        q = c.empty(x->sizes(), out);
        s = c.empty({B, S}, Dt::Float);
        return q8k_norm_modulate_quant(cptr(x), cptr(sc), cptr(sh), q.data_ptr(), dt_code(out), s.data_ptr<float>(), B * S,
                                       (int)dim, S, scale, c.stream());
    });
    return launched(rc, "norm_modulate_quant") ? list2(std::move(q), std::move(s)) : nullptr;
    FAST_END
}

// transpose_quant(x, row_scales | None)
PyObject* transpose_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 2);
    const at::Tensor* x = c.tensor(0);
    const at::Tensor* rs = c.optional(1, Dt::Float);
    OR_NONE(c);
    c.need(x->dim() == 2 && int_sized(x->size(0)) && int_sized(x->size(1)) && dt_code(x->scalar_type()) >= 0 &&
           (rs == nullptr || rs->numel() == x->size(0)));
    OR_NONE(c);
    const int64_t rows = x->size(0), k = x->size(1);
    at::Tensor q, s;
    const int rc = launch([&] {
        q = c.empty({k, rows}, Dt::Float8_e4m3fn);
        s = c.empty({k}, Dt::Float);
        return q8k_transpose_quant(cptr(x), dt_code(x->scalar_type()), fptr(rs), q.data_ptr(), s.data_ptr<float>(), (int)rows,
                                   (int)k, c.stream());
    });
    return launched(rc, "transpose_quant") ? list2(std::move(q), std::move(s)) : nullptr;
    FAST_END
}

// dequant_hadamard(x, row_scales, scale)
PyObject* dequant_hadamard(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 3);
    const at::Tensor* x = c.tensor(0, Dt::Char);
    const at::Tensor* rs = c.tensor(1, Dt::Float);
    const float scale = c.real(2);
    OR_NONE(c);
    c.need(x->dim() == 2 && int_sized(x->size(1)) && rs->numel() == x->size(0));
    OR_NONE(c);
    at::Tensor y;
    const int rc = launch([&] {
        y = c.empty(x->sizes(), Dt::BFloat16);
        return q8k_dequant_hadamard(cptr(x), fptr(rs), y.data_ptr(), x->size(0), (int)x->size(1), scale, c.stream());
    });
    return launched(rc, "dequant_hadamard") ? wrap(std::move(y)) : nullptr;
    FAST_END
}

// rms_norm(x, weights | None, out_type)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 3);
    const at::Tensor* x = c.tensor(0);
    const at::Tensor* w = c.optional(1, Dt::Float);
    OR_NONE(c);
    const Dt out = c.dtype(2, x->scalar_type());
    c.need(has_rows(x) && dt_code(x->scalar_type()) >= 0 && dt_code(out) >= 0 && (w == nullptr || w->numel() == x->size(-1)));
    OR_NONE(c);
    const int dim = (int)x->size(-1);
    at::Tensor y, r;
    const int rc = launch([&] {
        y = c.empty(x->sizes(), out);
        r = c.empty(lead(*x), Dt::Float);
        return q8k_rms_norm(cptr(x), dt_code(x->scalar_type()), fptr(w), y.data_ptr(), dt_code(out), r.data_ptr<float>(),
                            x->numel() / dim, dim, c.stream());
    });
    return launched(rc, "rms_norm") ? list2(std::move(y), std::move(r)) : nullptr;
    FAST_END
}

// rms_norm_backward(x_normed, x_norms, grad_out, weights | None, out_type)
PyObject* rms_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 5);
    const at::Tensor* y = c.tensor(0);
    const at::Tensor* r = c.tensor(1, Dt::Float);
    const at::Tensor* g = c.tensor(2);
    const at::Tensor* w = c.optional(3, Dt::Float);
    OR_NONE(c);
    const Dt out = c.dtype(4, y->scalar_type());
    c.need(has_rows(y) && dt_code(y->scalar_type()) >= 0 && dt_code(out) >= 0 && g->scalar_type() == out &&
           g->sizes() == y->sizes() && (w == nullptr || w->numel() == y->size(-1)));
    OR_NONE(c);
    const int dim = (int)y->size(-1);
    const int64_t rows = y->numel() / dim;
    c.need(r->numel() == rows);
    OR_NONE(c);
    at::Tensor gx;
    const int rc = launch([&] {
        gx = c.empty(y->sizes(), out);
        return q8k_rms_norm_backward(cptr(y), dt_code(y->scalar_type()), fptr(r), cptr(g), fptr(w), gx.data_ptr(), dt_code(out),
                                     rows, dim, c.stream());
    });
    return launched(rc, "rms_norm_backward") ? wrap(std::move(gx)) : nullptr;
    FAST_END
}

// rope(x, cos, sin, out_type) and rope_backward(grad, cos, sin, out_type)
using RopeFn = int (*)(const void*, int, const float*, const float*, void*, int, int64_t, int, int64_t, void*);
PyObject* rope_like(RopeFn fn, const char* op, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 4);
    const at::Tensor* x = c.tensor(0);
    const at::Tensor* co = c.tensor(1, Dt::Float);
    const at::Tensor* si = c.tensor(2, Dt::Float);
    OR_NONE(c);
    const Dt out = c.dtype(3, x->scalar_type());
    c.need(has_rows(x) && dt_code(x->scalar_type()) >= 0 && dt_code(out) >= 0 && co->sizes() == si->sizes() && co->dim() >= 1 &&
           co->size(-1) == x->size(-1));
    OR_NONE(c);
    const int dim = (int)x->size(-1);
    const int64_t rows = x->numel() / dim, table = co->numel() / dim;
    c.need(table > 0 && (table == rows || (rows % table == 0 && co->dim() == x->dim() && co->size(0) == 1)));
    OR_NONE(c);
    at::Tensor y;
    const int rc = launch([&] {
        y = c.empty(x->sizes(), out);
        return fn(cptr(x), dt_code(x->scalar_type()), fptr(co), fptr(si), y.data_ptr(), dt_code(out), rows, dim,
                  table == rows ? 0 : table, c.stream());
    });
    return launched(rc, op) ? wrap(std::move(y)) : nullptr;
    FAST_END
}
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) { return rope_like(q8k_rope, "rope", args, n); }
PyObject* rope_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return rope_like(q8k_rope_backward, "rope_backward", args, n);
}

// ---------------------------------------------------------------- products
// mm(a, b, bias | None, a_scales, b_scales, fuse_gelu, out_type, in_type, op): in_type int8 or e4m3, op the public name
PyObject* mm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 9);
    const Dt in = c.dtype(7, Dt::Undefined);
    const at::Tensor* a = c.tensor(0, in);
    const at::Tensor* b = c.tensor(1, in);
    const at::Tensor* bias = c.optional(2, Dt::Float);
    const at::Tensor* sa = c.tensor(3, Dt::Float);
    const at::Tensor* sb = c.tensor(4, Dt::Float);
    const bool gelu = c.flag(5);
    const Dt out = c.dtype(6, Dt::Float8_e4m3fn);
    c.need(c.ok && PyUnicode_Check(args[8]));
    OR_NONE(c);
    c.need(quant_type(in) && dt_code(out) >= 0 &&
           (a->dim() == 2 || a->dim() == 3) && (b->dim() == 2 || b->dim() == 3));
    OR_NONE(c);
    const int64_t ba = a->dim() == 3 ? a->size(0) : 1, m = a->size(-2), k = a->size(-1);
    const int64_t bb = b->dim() == 3 ? b->size(0) : 1, nn = b->size(-2);
    c.need(b->size(-1) == k && (ba == bb || ba == 1 || bb == 1) && int_sized(ba * m) && int_sized(bb * nn) && int_sized(k) &&
           sa->numel() == ba * m && sb->numel() == bb * nn && (bias == nullptr || bias->numel() == nn));
    int* word = c.status();
    OR_NONE(c);
    at::Tensor y;
    const bool i8 = in == Dt::Char;
    const int rc = launch([&] {
        y = c.empty({ba > bb ? ba : bb, m, nn}, out);
        return (i8 ? q8k_q8_mm : q8k_fp8_mm)(cptr(a), cptr(b), fptr(bias), fptr(sa), fptr(sb), y.data_ptr(), dt_code(out), (int)ba,
                                             (int)bb, (int)m, (int)nn, (int)k, gelu, word, c.stream());
    });
    const char* op = rc == Q8K_OK ? "" : PyUnicode_AsUTF8(args[8]);
    return op != nullptr && launched(rc, op) ? wrap(std::move(y)) : nullptr;
    FAST_END
}

// mm_gate_residual(a, b, bias | None, a_scales, b_scales, gate | None, resid)
PyObject* mm_gate_residual(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* a = c.tensor(0);
    const at::Tensor* b = c.tensor(1);
    const at::Tensor* bias = c.optional(2, Dt::Float);
    const at::Tensor* sa = c.tensor(3, Dt::Float);
    const at::Tensor* sb = c.tensor(4, Dt::Float);
    const at::Tensor* gate = c.optional(5, Dt::BFloat16);
    const at::Tensor* resid = c.tensor(6, Dt::BFloat16);
    OR_NONE(c);
    c.need(quant_type(a->scalar_type()) && b->scalar_type() == a->scalar_type() && (a->dim() == 2 || a->dim() == 3) &&
           b->dim() == 2);
    OR_NONE(c);
    const int64_t ba = a->dim() == 3 ? a->size(0) : 1, m = a->size(-2), k = a->size(-1), nn = b->size(0);
    c.need(b->size(1) == k && int_sized(ba * m) && int_sized(nn) && int_sized(k) && sa->numel() == ba * m && sb->numel() == nn &&
           (bias == nullptr || bias->numel() == nn) && resid->numel() == ba * m * nn &&
           (gate == nullptr || gate->numel() == ba * nn));
    int* word = c.status();
    OR_NONE(c);
    at::Tensor y;
    const int rc = launch([&] {
        y = c.empty({ba, m, nn}, Dt::BFloat16);
        return q8k_mm_gate_residual(a->scalar_type() == Dt::Char, cptr(a), cptr(b), fptr(bias), fptr(sa), fptr(sb), cptr(gate),
                                    cptr(resid), gate == nullptr ? 1 : m, y.data_ptr(), (int)ba, 1, (int)m, (int)nn, (int)k, word,
                                    c.stream());
    });
    return launched(rc, "mm_gate_residual") ? wrap(std::move(y)) : nullptr;
    FAST_END
}

// linear(x, w, w_scales, bias | None, use_hadamard, fuse_gelu, out_type)
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* x = c.tensor(0);
    const at::Tensor* w = c.tensor(1);
    const at::Tensor* ws = c.tensor(2, Dt::Float);
    const at::Tensor* bias = c.optional(3, Dt::Float);
    const bool had = c.flag(4), gelu = c.flag(5);
    const Dt out = c.dtype(6, Dt::Undefined);
    OR_NONE(c);
    c.need((x->dim() == 2 || x->dim() == 3) && w->dim() == 2 && quant_type(w->scalar_type()) && dt_code(x->scalar_type()) >= 0 &&
           dt_code(out) >= 0 && has_rows(x) && w->size(1) == x->size(-1) && int_sized(w->size(0)) && ws->numel() == w->size(0) &&
           (bias == nullptr || bias->numel() == w->size(0)));
    int* word = c.status();
    OR_NONE(c);
    const int64_t k = x->size(-1), m = x->numel() / k, nn = w->size(0);
    c.need(int_sized(m));
    OR_NONE(c);
    // Scratch for the quantised rows, given back to the allocator when the call returns: it is handed out again only to
    // work that is queued behind these kernels on the same stream.
    const size_t need = q8k_linear_workspace_bytes((int)m, (int)k);
    at::Tensor scratch, y;
    const int rc = launch([&] {
        scratch = c.empty({(int64_t)(need > 0 ? need : 1)}, Dt::Byte);
        y = x->dim() == 3 ? c.empty({x->size(0), x->size(1), nn}, out) : c.empty({1, m, nn}, out);
        return q8k_linear(cptr(x), dt_code(x->scalar_type()), cptr(w), dt_code(w->scalar_type()), fptr(ws), fptr(bias),
                          y.data_ptr(), dt_code(out), (int)m, (int)nn, (int)k, had, gelu, scratch.data_ptr(), need, word, c.stream());
    });
    return launched(rc, "linear") ? wrap(std::move(y)) : nullptr;
    FAST_END
}

// ---------------------------------------------------------------- attention
// flash_attention(q, k, v, scale, key_lens | None, out_type, token_major): v as rows [B,H,N,64]
PyObject* flash_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* q = c.tensor(0, Dt::Float8_e4m3fn);
    const at::Tensor* k = c.tensor(1, Dt::Float8_e4m3fn);
    const at::Tensor* v = c.tensor(2, Dt::Float8_e4m3fn);
    const float scale = c.real(3);
    const at::Tensor* lens = c.optional(4, Dt::Int);
    const Dt out = c.dtype(5, Dt::Float8_e4m3fn);
    const bool token_major = c.flag(6);
    OR_NONE(c);
    c.need(q->dim() == 4 && k->dim() == 4 && v->sizes() == k->sizes() && dt_code(out) >= 0);
    OR_NONE(c);
    const int64_t B = q->size(0), H = q->size(1), M = q->size(2), N = k->size(2);
    c.need(q->size(3) == 64 && k->size(3) == 64 && k->size(0) == B && k->size(1) == H && int_sized(B) && int_sized(H) &&
           int_sized(M) && int_sized(N) && (lens == nullptr || (lens->dim() == 1 && lens->size(0) == B)));
    int* word = c.status();
    OR_NONE(c);
    at::Tensor o;
    const int rc = launch([&] {
        o = token_major ? c.empty({B, M, H, 64}, out) : c.empty({B, H, M, 64}, out);
        void* outs[1] = {o.data_ptr()};
        return q8k_flash_attention_v_rows(cptr(q), cptr(k), cptr(v), outs, 1, dt_code(out), (int)B, (int)H, (int)M, (int)N,
                                          H * M * 64, token_major ? 64 : M * 64, token_major ? H * 64 : 64, scale,
                                          static_cast<const int*>(cptr(lens)), word, c.stream());
    });
    if (!launched(rc, "flash_attention")) return nullptr;
    return wrap(token_major ? o.transpose(1, 2) : std::move(o));
    FAST_END
}

// attention_prep_rows(q, k, v, apply_hadamard, scale): [B,H,S,64] views of any batch, head and token strides
PyObject* attention_prep_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 5);
    const at::Tensor* t[3];
    for (int i = 0; i < 3; ++i) t[i] = c.tensor(i, Dt::BFloat16, true);
    const bool had = c.flag(3);
    const float scale = c.real(4);
    OR_NONE(c);
    for (int i = 0; i < 3; ++i)
        c.need(t[i]->dim() == 4 && t[i]->size(3) == 64 && t[i]->stride(3) == 1 && t[i]->stride(0) % 8 == 0 &&
               t[i]->stride(1) % 8 == 0 && t[i]->stride(2) % 8 == 0 && (uintptr_t)cptr(t[i]) % 16 == 0 && int_sized(t[i]->size(2)));
    OR_NONE(c);
    const int64_t B = t[0]->size(0), H = t[0]->size(1);
    c.need(t[1]->size(0) == B && t[1]->size(1) == H && t[2]->sizes() == t[1]->sizes() && int_sized(B) && int_sized(H));
    OR_NONE(c);
    at::Tensor o[3];
    const int rc = launch([&] {
        for (int i = 0; i < 3; ++i) o[i] = c.empty({B, H, t[i]->size(2), 64}, Dt::Float8_e4m3fn);
        return q8k_attention_prep_rows(cptr(t[0]), cptr(t[1]), cptr(t[2]), o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(),
                                       (int)B, (int)H, (int)t[0]->size(2), (int)t[1]->size(2), t[0]->stride(0), t[0]->stride(2),
                                       t[0]->stride(1), t[1]->stride(0), t[1]->stride(2), t[1]->stride(1), t[2]->stride(0),
                                       t[2]->stride(2), t[2]->stride(1), had, scale, c.stream());
    });
    if (!launched(rc, "attention_prep_rows")) return nullptr;
    return tuple_of(o);
    FAST_END
}

// The pre-passes of a projection's output.  Q, K and V (those that an op has) are column slices [B,S,H*64] of one tensor; the
// result is their e4m3 tensors.
struct Prep {
    const at::Tensor *q = nullptr, *k = nullptr, *v = nullptr, *wq = nullptr, *wk = nullptr;
    at::Tensor cos, sin;                                       // owned: a list may change while the lock is given up
    int64_t heads = 0;
    bool hadamard = false;
    float scale = 0.f;
    bool rotate = false;

    // freqs_cis: None or a (cos, sin) tuple or list; anything else is left as it is, an iterator unread
    void tables(Call& c, int i) {
        if (!c.ok || c.args[i] == Py_None) return;
        PyObject* f = c.args[i];
        if (!(PyTuple_CheckExact(f) || PyList_CheckExact(f)) || PySequence_Fast_GET_SIZE(f) != 2) { c.ok = false; return; }
        const at::Tensor* t[2] = {nullptr, nullptr};
        for (int k = 0; k < 2 && c.ok; ++k) t[k] = c.tensor_of(PySequence_Fast_GET_ITEM(f, k));
        c.need(c.ok && t[0]->scalar_type() == Dt::Float && t[1]->scalar_type() == Dt::Float);
        if (!c.ok) return;
        cos = *t[0];
        sin = *t[1];
        rotate = true;
    }
};

PyObject* prep(Call& c, const Prep& a, const char* op) {
    OR_NONE(c);
    const at::Tensor& k = *a.k;
    const at::Tensor* x[3] = {a.q, a.k, a.v};
    c.need(k.dim() == 3 && k.size(2) == a.heads * 64);
    OR_NONE(c);
    const int64_t B = k.size(0), S = k.size(1), C = a.heads * 64, rs = k.stride(1);
    for (const at::Tensor* t : x)
        c.need(t == nullptr || (t->sizes() == k.sizes() && t->strides() == k.strides() && (uintptr_t)cptr(t) % 16 == 0));
    c.need(k.stride(2) == 1 && k.stride(0) == S * rs && rs % 8 == 0 && int_sized(B) && int_sized(S) && int_sized(C) &&
           a.wk->numel() == C && (a.wq == nullptr || a.wq->numel() == C) &&
           (!a.rotate || (a.cos.numel() == S * C && a.sin.numel() == S * C)));
    OR_NONE(c);
    const float* co = a.rotate ? fptr(&a.cos) : nullptr;
    const float* si = a.rotate ? fptr(&a.sin) : nullptr;
    at::Tensor o[3];
    void* p[3] = {nullptr, nullptr, nullptr};
    const int rc = launch([&] {
        for (int i = 0; i < 3; ++i)
            if (x[i] != nullptr) {
                o[i] = c.empty({B, a.heads, S, 64}, Dt::Float8_e4m3fn);
                p[i] = o[i].data_ptr();
            }
        if (a.v != nullptr)
            return q8k_qkv_prep(cptr(a.q), cptr(a.k), cptr(a.v), rs, fptr(a.wq), fptr(a.wk), co, si, p[0], p[1], p[2], (int)B,
                                (int)S, (int)a.heads, a.hadamard, a.scale, c.stream());
        if (a.q != nullptr)
            return q8k_qk_norm_rope_prep_pair(cptr(a.q), cptr(a.k), rs, fptr(a.wq), fptr(a.wk), co, si, p[0], p[1], (int)B, (int)S,
                                              (int)a.heads, a.hadamard, a.scale, c.stream());
        return q8k_qk_norm_rope_prep(cptr(a.k), rs, fptr(a.wk), co, si, p[1], (int)B, (int)S, (int)a.heads, a.hadamard, a.scale,
                                     c.stream());
    });
    if (!launched(rc, op)) return nullptr;
    return a.q == nullptr && a.v == nullptr ? wrap(std::move(o[1])) : tuple_of(o);
}

// qk_norm_rope_prep(x, norm_w, freqs_cis, heads, apply_hadamard, scale)
PyObject* qk_norm_rope_prep(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 6);
    Prep a;
    a.k = c.tensor(0, Dt::BFloat16, true);
    a.wk = c.tensor(1, Dt::Float);
    a.tables(c, 2);
    a.heads = c.integer(3);
    a.hadamard = c.flag(4);
    a.scale = c.real(5);
    return prep(c, a, "qk_norm_rope_prep");
    FAST_END
}

// kv_prep(xk, xv, norm_wk, heads, apply_hadamard, scale)
PyObject* kv_prep(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 6);
    Prep a;
    a.k = c.tensor(0, Dt::BFloat16, true);
    a.v = c.tensor(1, Dt::BFloat16, true);
    a.wk = c.tensor(2, Dt::Float);
    a.heads = c.integer(3);
    a.hadamard = c.flag(4);
    a.scale = c.real(5);
    return prep(c, a, "qkv_prep");
    FAST_END
}

// qk_norm_rope_prep_pair(xq, xk, norm_wq, norm_wk, freqs_cis, heads, apply_hadamard, scale, xv | None)
PyObject* qk_norm_rope_prep_pair(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 9);
    Prep a;
    a.q = c.tensor(0, Dt::BFloat16, true);
    a.k = c.tensor(1, Dt::BFloat16, true);
    a.wq = c.tensor(2, Dt::Float);
    a.wk = c.tensor(3, Dt::Float);
    a.tables(c, 4);
    a.heads = c.integer(5);
    a.hadamard = c.flag(6);
    a.scale = c.real(7);
    if (c.ok && args[8] != Py_None) a.v = c.tensor(8, Dt::BFloat16, true);
    return prep(c, a, a.v == nullptr ? "qk_norm_rope_prep_pair" : "qkv_prep");
    FAST_END
}

// ---------------------------------------------------------------- layer norm, rotary positions, gated projection, head norm, 4-bit linear
// These are differentiable: where an input has a gradient the call leaves a node of torch's C++ autograd behind, whose backward pass
// launches without the interpreter.  (A Python autograd.Function costs some 60 us of host time for one forward and backward pass, the
// kernels of a short call 10.)  What functional.layer_norm.layer_norm, functional.rotary, functional.gated, functional.head_norm and functional.fp4 do with tensors
// that these do not take is the same.  The underscore marks them: they answer for functions of functional/, not of native.py.

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int type_code(Dt t) { return t == Dt::Half ? Q8K_DT_F16 : dt_code(t); }      // (the ops above leave fp16 to their Python bodies)

// An argument that may be missing.  (apply() does not take undefined tensors; the inputs that it numbers are those that are there.)
using Maybe = std::optional<at::Tensor>;
Maybe maybe(const at::Tensor* t) { return t == nullptr ? Maybe() : Maybe(*t); }
at::Tensor value(const Maybe& t) { return t.has_value() ? *t : at::Tensor(); }

struct Refused { int rc; const char* op; };                    // a launch's error on its way to Q8KernelError

void must(int rc, const char* op) {
    if (rc != Q8K_OK) throw Refused{rc, op};
}
// In a backward pass, which autograd runs: its error becomes a RuntimeError.
void must_backward(int rc, const char* op) {
    if (rc != Q8K_OK) throw std::runtime_error(std::string(op) + ": " + q8k_error_string(rc) + ": " + q8k_last_error_detail());
}
template <typename F> PyObject* answer(F&& f) {                // f() -> PyObject*, with Refused turned into the Python error
    try {
        return f();
    } catch (const Refused& e) {
        if (launched(e.rc, e.op)) Py_RETURN_NONE;
        return nullptr;
    }
}
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
at::Tensor empty_like_dtype(at::IntArrayRef shape, const at::Tensor& like, Dt type) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}
float* out_f(at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const at::Tensor* defined(const at::Tensor& t) { return t.defined() ? &t : nullptr; }
bool wants_grad(const at::Tensor* t) { return t != nullptr && t->requires_grad(); }
// Carries a forward-mode derivative (there is one level of them), which the Python bodies refuse.
bool has_tangent(const at::Tensor* t) { return t != nullptr && t->_fw_grad(0).defined(); }

// Gradients that cannot be differentiated again say so when that is tried, as once_differentiable does in Python.
variable_list once_only(variable_list&& grads, const variable_list& incoming) {
    bool graph = false;
    for (const Variable& g : incoming) graph = graph || (g.defined() && g.requires_grad());
    if (!c10::GradMode::is_enabled() || !graph) return std::move(grads);
    for (Variable& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that is differentiable once",
                                                                 (int)grads.size());
    return error->apply(std::move(grads));
}

// ---- _layer_norm(x, weight | None, bias | None, eps, out_type)
struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Variable run(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, double eps, Dt out, at::Tensor* mean, at::Tensor* rstd) {
        const int dim = (int)x.size(-1);
        at::Tensor y = empty_like_dtype(x.sizes(), x, out);
        if (mean != nullptr) {
            *mean = empty_like_dtype(lead(x), x, Dt::Float);
            *rstd = empty_like_dtype(lead(x), x, Dt::Float);
        }
        must(q8k_layer_norm(x.const_data_ptr(), type_code(x.scalar_type()), dim, fptr(defined(w)), fptr(defined(b)), y.data_ptr(), type_code(out),
                            mean != nullptr ? mean->data_ptr<float>() : nullptr, rstd != nullptr ? rstd->data_ptr<float>() : nullptr,
                            x.numel() / dim, dim, (float)eps, stream_of(x)), "layer_norm");
        return y;
    }
    static Variable forward(AutogradContext* ctx, const Variable& x, const Maybe& w, const Maybe& b, double eps, int64_t out) {
        at::Tensor mean, rstd;
        Variable y = run(x, value(w), value(b), eps, (Dt)out, &mean, &rstd);
        ctx->save_for_backward({x, value(w), mean, rstd});
        ctx->saved_data["bias"] = b.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(5);
        if (!grads[0].defined()) return result;
        {
            at::NoGradGuard no_grad;
            const at::Tensor &x = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
            at::Tensor g = grads[0];
            if (g.scalar_type() == Dt::Float8_e4m3fn) g = g.to(Dt::BFloat16);       // exact
            g = g.contiguous();
            const int dim = (int)x.size(-1);
            const int64_t rows = x.numel() / dim;
            at::Tensor dx, dw, db, work;
            if (ctx->needs_input_grad(0)) dx = empty_like_dtype(x.sizes(), x, x.scalar_type());
            const bool has_w = w.defined();
            if (has_w && ctx->needs_input_grad(1)) dw = empty_like_dtype({dim}, x, Dt::Float);
            if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1 + has_w)) db = empty_like_dtype({dim}, x, Dt::Float);
            int64_t bytes = 0;
            if (dw.defined() || db.defined()) {
                bytes = (int64_t)q8k_layer_norm_backward_workspace_bytes(rows, dim);
                work = empty_like_dtype({bytes}, x, Dt::Byte);
            }
            must_backward(q8k_layer_norm_backward(x.const_data_ptr(), type_code(x.scalar_type()), dim, g.const_data_ptr(),
                                                  type_code(g.scalar_type()), mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(),
                                                  fptr(defined(w)), dx.defined() ? dx.data_ptr() : nullptr, out_f(dw), out_f(db), rows, dim,
                                                  work.defined() ? work.data_ptr() : nullptr, (size_t)bytes, stream_of(x)),
                          "layer_norm_backward");
            result[0] = dx;
            result[1] = dw;
            result[2] = db;
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 5);
    const at::Tensor* x = c.tensor(0);
    const at::Tensor* w = c.optional(1, Dt::Float);
    const at::Tensor* b = c.optional(2, Dt::Float);
    const float eps = c.real(3);
    OR_NONE(c);
    const Dt in = x->scalar_type(), out = c.dtype(4, in);
    c.need(has_rows(x) && x->size(-1) <= 16384 && int_sized(x->numel() / x->size(-1)) &&
           ((in == out && (in == Dt::Float || in == Dt::Half || in == Dt::BFloat16)) || (in == Dt::BFloat16 && out == Dt::Float8_e4m3fn) ||
            (in == Dt::Float && (out == Dt::BFloat16 || out == Dt::Half))));
    OR_NONE(c);
    for (const at::Tensor* v : {w, b}) c.need(v == nullptr || (v->dim() == 1 && v->size(0) == x->size(-1)));
    c.need(!has_tangent(x) && !has_tangent(w) && !has_tangent(b));
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        at::Tensor y;
        {
            WithoutGil unlocked;
            if (c10::GradMode::is_enabled() && (x->requires_grad() || wants_grad(w) || wants_grad(b)))
                y = LayerNormNode::apply(*x, maybe(w), maybe(b), (double)eps, (int64_t)out);
            else
                y = LayerNormNode::run(*x, value(maybe(w)), value(maybe(b)), eps, out, nullptr, nullptr);
        }
        return wrap(std::move(y));
    });
    FAST_END
}

// ---- _rotary(q, k | None, positions | None, frequencies, amplitude, half): frequencies as float64, or their bits as int64, which is how
// RotaryEmbedding holds them (a view as float64 would cost as much as the launch)
struct RotaryNode : torch::autograd::Function<RotaryNode> {
    // q and k of [batch, seq, heads, dim], or without the batch; either may be undefined
    static variable_list run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& freq, double amplitude, bool half,
                             bool backward, int& rc) {
        const at::Tensor& x = q.defined() ? q : k;
        const int64_t d = x.dim(), batch = d == 4 ? x.size(0) : 1, seq = x.size(d - 3), dim = x.size(d - 1);
        variable_list out(2);
        int64_t stride[2][2][3] = {};
        const at::Tensor* in[2] = {&q, &k};
        for (int i = 0; i < 2; ++i) {
            if (!in[i]->defined()) continue;
            out[i] = empty_like_dtype(in[i]->sizes(), x, x.scalar_type());
            for (int j = 0; j < 2; ++j) {
                const at::Tensor& t = j == 0 ? *in[i] : out[i];
                stride[i][j][0] = d == 4 ? t.stride(0) : 0;
                stride[i][j][1] = t.stride(d - 3);
                stride[i][j][2] = t.stride(d - 2);
            }
        }
        const int64_t pb = pos.defined() && pos.dim() == 2 && pos.size(0) > 1 ? pos.stride(0) : 0;
        const int64_t pt = pos.defined() ? pos.stride(-1) : 0;
        auto heads = [&](const at::Tensor& t) { return t.defined() ? (int)t.size(d - 2) : 0; };
        rc = q8k_rotary(cptr(defined(q)), stride[0][0], out[0].defined() ? out[0].data_ptr() : nullptr, stride[0][1], heads(q), cptr(defined(k)),
                        stride[1][0], out[1].defined() ? out[1].data_ptr() : nullptr, stride[1][1], heads(k), type_code(x.scalar_type()),
                        cptr(defined(pos)), pos.defined() && pos.scalar_type() == Dt::Long, pb, pt, static_cast<const double*>(freq.const_data_ptr()),
                        (float)amplitude, (int)batch, (int)seq, (int)dim, (int)(2 * freq.numel()), half, backward, stream_of(x));
        return out;
    }
    static variable_list forward(AutogradContext* ctx, const Variable& q, const Maybe& k, const Maybe& pos, const Variable& freq,
                                 double amplitude, bool half) {
        int rc = 0;
        variable_list out = run(q, value(k), value(pos), freq, amplitude, half, false, rc);
        must(rc, "rotary");
        ctx->save_for_backward({value(pos), freq});
        ctx->saved_data["amplitude"] = amplitude;
        ctx->saved_data["half"] = half;
        ctx->set_materialize_grads(false);
        if (!k.has_value()) out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(6);
        {
            at::NoGradGuard no_grad;
            at::Tensor g[2];
            for (size_t i = 0; i < grads.size(); ++i) {
                if (!grads[i].defined() || !ctx->needs_input_grad(i)) continue;
                g[i] = grads[i].stride(-1) == 1 ? grads[i] : grads[i].contiguous();
            }
            if (!g[0].defined() && !g[1].defined()) return result;
            int rc = 0;
            variable_list d = run(g[0], g[1], saved[0], saved[1], ctx->saved_data["amplitude"].toDouble(), ctx->saved_data["half"].toBool(),
                                  true, rc);
            must_backward(rc, "rotary");
            result[0] = d[0];
            result[1] = d[1];
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 6);
    const at::Tensor* q = c.tensor(0, true);
    const at::Tensor* k = c.ok && args[1] != Py_None ? c.tensor(1, true) : nullptr;
    const at::Tensor* pos = c.ok && args[2] != Py_None ? c.tensor(2, true) : nullptr;
    const at::Tensor* freq = c.tensor(3);
    const float amplitude = c.real(4);
    const bool half = c.flag(5);
    OR_NONE(c);
    const Dt t = q->scalar_type();
    const int64_t d = q->dim();
    c.need((freq->scalar_type() == Dt::Double || freq->scalar_type() == Dt::Long) && (t == Dt::BFloat16 || t == Dt::Half || t == Dt::Float) &&
           (d == 3 || d == 4) && q->stride(-1) == 1 && freq->dim() == 1);
    OR_NONE(c);
    const int64_t batch = d == 4 ? q->size(0) : 1, seq = q->size(d - 3), dim = q->size(-1);
    c.need(int_sized(batch) && int_sized(seq) && dim <= 4096 && freq->numel() >= 1 && 2 * freq->numel() <= dim && q->size(d - 2) <= 65536);
    if (k != nullptr) {
        c.need(k->scalar_type() == t && k->dim() == d && k->stride(-1) == 1 && k->size(-1) == dim && k->size(d - 3) == seq &&
               (d == 3 || k->size(0) == batch) && k->size(d - 2) <= 65536);
    }
    if (pos != nullptr) {
        c.need((pos->scalar_type() == Dt::Long || pos->scalar_type() == Dt::Int) && (pos->dim() == 1 || pos->dim() == 2) &&
               pos->size(-1) == seq && (pos->dim() == 1 || pos->size(0) == 1 || pos->size(0) == batch));
    }
    OR_NONE(c);
    c.need((q->size(d - 2) + (k != nullptr ? k->size(d - 2) : 0)) * dim <= (1 << 24) && !has_tangent(q) && !has_tangent(k) &&
           !has_tangent(freq));
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        variable_list out;
        {
            WithoutGil unlocked;
            if (c10::GradMode::is_enabled() && (q->requires_grad() || wants_grad(k))) {
                out = RotaryNode::apply(*q, maybe(k), maybe(pos), *freq, (double)amplitude, half);
            } else {
                int rc = 0;
                out = RotaryNode::run(*q, value(maybe(k)), value(maybe(pos)), *freq, amplitude, half, false, rc);
                must(rc, "rotary");
            }
        }
        PyObject* r = PyTuple_New(2);
        if (r == nullptr) return nullptr;
        PyTuple_SET_ITEM(r, 0, wrap(std::move(out[0])));
        if (k != nullptr) {
            PyTuple_SET_ITEM(r, 1, wrap(std::move(out[1])));
        } else {
            Py_INCREF(Py_None);
            PyTuple_SET_ITEM(r, 1, Py_None);
        }
        return r;
    });
    FAST_END
}

// ---- _gated_linear(a, b, bias | None, scale_b, activation code, int8, rotate)
struct GatedNode : torch::autograd::Function<GatedNode> {
    static at::Tensor run(const at::Tensor& a, const at::Tensor& b, const at::Tensor& bias, const at::Tensor& scale, int act, bool rotate,
                          at::Tensor* pre) {
        const int64_t k = b.size(1), f = b.size(0) / 2, m = a.numel() / k;
        at::DimVector shape(lead(a).begin(), lead(a).end());
        const int64_t bytes = (int64_t)q8k_gated_linear_workspace_bytes((int)m, (int)k);
        at::Tensor work = empty_like_dtype({bytes}, a, Dt::Byte);
        shape.push_back(f);
        at::Tensor out = empty_like_dtype(shape, a, Dt::BFloat16);
        if (pre != nullptr) {
            shape.back() = 2;
            shape.push_back(f);
            *pre = empty_like_dtype(shape, a, Dt::BFloat16);
        }
        must(q8k_gated_linear(a.const_data_ptr(), type_code(a.scalar_type()), b.const_data_ptr(), type_code(b.scalar_type()),
                              scale.const_data_ptr<float>(), fptr(defined(bias)), out.data_ptr(), pre != nullptr ? pre->data_ptr() : nullptr, act,
                              (int)m, (int)f, (int)k, rotate, work.data_ptr(), (size_t)bytes, g_status[a.device().index()]->data_ptr<int>(),
                              stream_of(a)), "gated_linear");
        return out;
    }
    static Variable forward(AutogradContext* ctx, const Variable& a, const Variable& b, const Maybe& bias, const Variable& scale, int64_t act,
                            bool rotate) {
        at::Tensor pre;
        Variable out = run(a, b, value(bias), scale, (int)act, rotate, &pre);
        ctx->save_for_backward({pre, b, scale});
        ctx->saved_data["act"] = act;
        ctx->saved_data["rotate"] = rotate;
        ctx->saved_data["type"] = (int64_t)a.scalar_type();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(6);
        if (!grads[0].defined()) return result;
        {
            at::NoGradGuard no_grad;
            const at::Tensor &pre = saved[0], &b = saved[1], &scale = saved[2];
            at::Tensor g = grads[0].to(Dt::BFloat16).contiguous();
            if (reinterpret_cast<uintptr_t>(g.const_data_ptr()) % 16 != 0) g = g.clone();
            const int64_t k = b.size(1), n = b.size(0), f = n / 2, m = g.numel() / f;
            at::DimVector shape(lead(g).begin(), lead(g).end());
            shape.push_back(k);
            at::Tensor dx = empty_like_dtype(shape, g, Dt::BFloat16);
            if (m > 0) {
                void* st = stream_of(g);
                int* word = g_status[g.device().index()]->data_ptr<int>();
                auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
                const int64_t work_bytes = up((int64_t)q8k_gated_weight_operand_workspace_bytes((int)f, (int)k));
                // one scratch: gradient rows and scales, weight operand and scales, its workspace, the product before the rotation
                const bool rotate = ctx->saved_data["rotate"].toBool();
                const int64_t at_gs = up(m * n), at_w = at_gs + up(4 * m), at_ws = at_w + up(k * n), at_work = at_ws + up(4 * k),
                              at_y = at_work + work_bytes, end = at_y + (rotate ? 2 * m * k : 0);
                at::Tensor scratch = empty_like_dtype({end}, g, Dt::Byte);
                uint8_t* s = static_cast<uint8_t*>(scratch.data_ptr());
                float *gs = reinterpret_cast<float*>(s + at_gs), *ws = reinterpret_cast<float*>(s + at_ws);
                must_backward(q8k_gated_backward_quant(g.const_data_ptr(), pre.const_data_ptr(), s, gs, (int)ctx->saved_data["act"].toInt(), (int)m,
                                                       (int)f, st), "gated_backward_quant");
                must_backward(q8k_gated_weight_operand(b.const_data_ptr(), type_code(b.scalar_type()), scale.const_data_ptr<float>(), s + at_w, ws,
                                                       (int)f, (int)k, s + at_work, (size_t)work_bytes, st), "gated_weight_operand");
                void* y = rotate ? static_cast<void*>(s + at_y) : dx.data_ptr();
                must_backward(q8k_fp8_mm(s, s + at_w, nullptr, gs, ws, y, Q8K_DT_BF16, 1, 1, (int)m, (int)k, (int)n, 0, word, st), "fp8_mm");
                if (rotate)
                    must_backward(q8k_fast_hadamard_transform(y, Q8K_DT_BF16, dx.data_ptr(), Q8K_DT_BF16, m, (int)k, k,
                                                              (float)(1.0 / std::sqrt((double)k)), st), "fast_hadamard_transform");
            }
            result[0] = dx.to((Dt)ctx->saved_data["type"].toInt());
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _gated_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* a = c.tensor(0);
    const at::Tensor* b = c.tensor(1);
    const at::Tensor* bias = c.optional(2, Dt::Float);
    const at::Tensor* scale = c.tensor(3, Dt::Float);
    const long act = c.integer(4);
    const bool int8 = c.flag(5), rotate = c.flag(6);
    OR_NONE(c);
    auto aligned = [](const at::Tensor* t) { return reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0; };
    c.need(aligned(a) && aligned(b) && (act == Q8K_ACT_SILU || act == Q8K_ACT_GELU_TANH) &&
           (a->scalar_type() == Dt::BFloat16 || (int8 && a->scalar_type() == Dt::Float8_e4m3fn)) && has_rows(a) && b->scalar_type() == (int8 ? Dt::Char : Dt::Float8_e4m3fn) && b->dim() == 2 && b->size(1) == a->size(-1));
    OR_NONE(c);
    const int64_t k = b->size(1), nn = b->size(0), m = a->numel() / k;
    const bool training = c10::GradMode::is_enabled() && a->requires_grad();
    c.need(nn > 0 && nn % 32 == 0 && nn <= 0x3fffffff && k % 16 == 0 && k <= 16384 && m <= 0x7fffff00 && scale->numel() == nn &&
           (bias == nullptr || bias->numel() == nn) && !(training && nn > 2 * 16384) && !has_tangent(a) &&
           !has_tangent(bias) && !has_tangent(scale));
    c.status();
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        at::Tensor out;
        {
            WithoutGil unlocked;
            out = training ? GatedNode::apply(*a, *b, maybe(bias), *scale, (int64_t)act, rotate)
                           : GatedNode::run(*a, *b, value(maybe(bias)), *scale, (int)act, rotate, nullptr);
        }
        return wrap(std::move(out));
    });
    FAST_END
}

// ---- rotation by positions of several axes, head norms
int position_code(Dt t) {
    switch (t) {
        case Dt::Int: return Q8K_POS_I32;
        case Dt::Long: return Q8K_POS_I64;
        case Dt::Float: return Q8K_POS_F32;
        case Dt::Double: return Q8K_POS_F64;
        default: return 0;
    }
}

// [batch, seq, heads, dim] or [seq, heads, dim]
struct HeadShape {
    int64_t d, batch, seq, dim;
    explicit HeadShape(const at::Tensor& x) : d(x.dim()), batch(d == 4 ? x.size(0) : 1), seq(x.size(d - 3)), dim(x.size(d - 1)) {}
    int heads(const at::Tensor& t) const { return t.defined() ? (int)t.size(d - 2) : 0; }
    void strides(const at::Tensor& t, int64_t (&s)[3]) const {
        if (!t.defined()) return;
        s[0] = d == 4 ? t.stride(0) : 0;
        s[1] = t.stride(d - 3);
        s[2] = t.stride(d - 2);
    }
};
const void* dense_ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Positions, frequencies and axes as a kernel takes them; axes undefined: one axis, positions undefined: 0, 1, ...
struct AngleArgs {
    const void* pos;
    int kind = Q8K_POS_I64, n_axes = 1;
    int64_t stride[3] = {0, 0, 0};
    const int* axes;
    const double* freq;
    int rotary_dim;
    AngleArgs(const at::Tensor& p, const at::Tensor& f, const at::Tensor& a)
        : pos(dense_ptr(p)), axes(static_cast<const int*>(dense_ptr(a))), freq(static_cast<const double*>(dense_ptr(f))),
          rotary_dim(f.defined() ? (int)(2 * f.numel()) : 0) {
        if (!p.defined()) return;
        kind = position_code(p.scalar_type());
        const bool several = a.defined();
        const int64_t d = p.dim(), token = several ? d - 2 : d - 1;
        if (token == 1 && p.size(0) > 1) stride[0] = p.stride(0);
        stride[1] = p.stride(token);
        if (several) {
            stride[2] = p.stride(d - 1);
            n_axes = (int)p.size(d - 1);
        }
    }
};

// What the fast path takes of queries, keys and their angles (freq may be null: no rotation).
void need_heads(Call& c, const at::Tensor* q, const at::Tensor* k, int64_t max_dim) {
    if (!c.ok) return;
    const Dt t = q->scalar_type();
    const int64_t d = q->dim();
    c.need((t == Dt::BFloat16 || t == Dt::Half || t == Dt::Float) && (d == 3 || d == 4) && q->stride(-1) == 1);
    if (!c.ok) return;
    const HeadShape s(*q);
    c.need(int_sized(s.batch) && int_sized(s.seq) && s.dim >= 1 && s.dim <= max_dim && q->size(d - 2) <= 65536);
    if (k != nullptr) {
        c.need(k->scalar_type() == t && k->dim() == d && k->stride(-1) == 1 && k->size(-1) == s.dim && k->size(d - 3) == s.seq &&
               (d == 3 || k->size(0) == s.batch) && k->size(d - 2) <= 65536);
    }
    if (!c.ok) return;
    c.need((q->size(d - 2) + (k != nullptr ? k->size(d - 2) : 0)) * s.dim <= (1 << 24) && !has_tangent(q) && !has_tangent(k));
}
void need_angles(Call& c, const at::Tensor* q, const at::Tensor* pos, const at::Tensor* freq, const at::Tensor* axes) {
    if (!c.ok) return;
    const HeadShape s(*q);
    c.need((freq != nullptr || (pos == nullptr && axes == nullptr)) && (axes == nullptr || pos != nullptr));
    if (!c.ok || freq == nullptr) return;
    c.need((freq->scalar_type() == Dt::Double || freq->scalar_type() == Dt::Long) && freq->dim() == 1 && freq->numel() >= 1 &&
           2 * freq->numel() <= s.dim && (axes == nullptr || (axes->dim() == 1 && axes->numel() == freq->numel())) && !has_tangent(freq) &&
           !has_tangent(pos));
    if (!c.ok || pos == nullptr) return;
    const int64_t last = axes != nullptr ? pos->dim() - 1 : pos->dim();          // dims before the axes
    const int code = position_code(pos->scalar_type());
    c.need((last == 1 || last == 2) && (axes != nullptr ? code != 0 && pos->size(-1) >= 1 && int_sized(pos->size(-1))
                                                        : code == Q8K_POS_I32 || code == Q8K_POS_I64));
    if (!c.ok) return;
    c.need(pos->size(last - 1) == s.seq && (last == 1 || pos->size(0) == 1 || pos->size(0) == s.batch));
}
PyObject* pair_of(variable_list&& out, bool both) {
    PyObject* r = PyTuple_New(2);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, wrap(std::move(out[0])));
    if (both) {
        PyTuple_SET_ITEM(r, 1, wrap(std::move(out[1])));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(r, 1, Py_None);
    }
    return r;
}
// A gradient with dense channels.
at::Tensor head_grad(const at::Tensor& g) { return g.stride(-1) == 1 || g.size(-1) == 1 ? g : g.contiguous(); }

// _axial_rotary(q, k | None, positions, frequencies, axes, amplitude, half): frequencies as for _rotary
struct AxialRotaryNode : torch::autograd::Function<AxialRotaryNode> {
    static variable_list run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& freq, const at::Tensor& axes,
                             double amplitude, bool half, bool backward, int& rc) {
        const at::Tensor& x = q.defined() ? q : k;
        const HeadShape s(x);
        const AngleArgs a(pos, freq, axes);
        variable_list out(2);
        int64_t in_s[2][3] = {}, out_s[2][3] = {};
        const at::Tensor* in[2] = {&q, &k};
        for (int i = 0; i < 2; ++i) {
            if (!in[i]->defined()) continue;
            out[i] = empty_like_dtype(in[i]->sizes(), x, x.scalar_type());
            s.strides(*in[i], in_s[i]);
            s.strides(out[i], out_s[i]);
        }
        rc = q8k_axial_rotary(dense_ptr(q), in_s[0], out_ptr(out[0]), out_s[0], s.heads(q), dense_ptr(k), in_s[1], out_ptr(out[1]), out_s[1],
                              s.heads(k), type_code(x.scalar_type()), a.pos, a.kind, a.stride, a.n_axes, a.axes, a.freq, (float)amplitude,
                              (int)s.batch, (int)s.seq, (int)s.dim, a.rotary_dim, half, backward, stream_of(x));
        return out;
    }
    static variable_list forward(AutogradContext* ctx, const Variable& q, const Maybe& k, const Variable& pos, const Variable& freq,
                                 const Variable& axes, double amplitude, bool half) {
        int rc = 0;
        variable_list out = run(q, value(k), pos, freq, axes, amplitude, half, false, rc);
        must(rc, "axial_rotary");
        ctx->save_for_backward({pos, freq, axes});
        ctx->saved_data["amplitude"] = amplitude;
        ctx->saved_data["half"] = half;
        ctx->set_materialize_grads(false);
        if (!k.has_value()) out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(7);
        {
            at::NoGradGuard no_grad;
            at::Tensor g[2];
            for (size_t i = 0; i < grads.size(); ++i)
                if (grads[i].defined() && ctx->needs_input_grad(i)) g[i] = head_grad(grads[i]);
            if (!g[0].defined() && !g[1].defined()) return result;
            int rc = 0;
            variable_list d = run(g[0], g[1], saved[0], saved[1], saved[2], ctx->saved_data["amplitude"].toDouble(),
                                  ctx->saved_data["half"].toBool(), true, rc);
            must_backward(rc, "axial_rotary");
            result[0] = d[0];
            result[1] = d[1];
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _axial_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* q = c.tensor(0, true);
    const at::Tensor* k = c.ok && args[1] != Py_None ? c.tensor(1, true) : nullptr;
    const at::Tensor* pos = c.tensor(2, true);
    const at::Tensor* freq = c.tensor(3);
    const at::Tensor* axes = c.tensor(4, Dt::Int);
    const float amplitude = c.real(5);
    const bool half = c.flag(6);
    need_heads(c, q, k, 4096);
    need_angles(c, q, pos, freq, axes);
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        variable_list out;
        {
            WithoutGil unlocked;
            if (c10::GradMode::is_enabled() && (q->requires_grad() || wants_grad(k))) {
                out = AxialRotaryNode::apply(*q, maybe(k), *pos, *freq, *axes, (double)amplitude, half);
            } else {
                int rc = 0;
                out = AxialRotaryNode::run(*q, value(maybe(k)), *pos, *freq, *axes, amplitude, half, false, rc);
                must(rc, "axial_rotary");
            }
        }
        return pair_of(std::move(out), k != nullptr);
    });
    FAST_END
}

// _head_norm(q, k | None, q_weight | None, k_weight | None, eps, positions | None, frequencies | None, axes | None, amplitude, half)
struct HeadNormNode : torch::autograd::Function<HeadNormNode> {
    static variable_list run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk, double eps, const at::Tensor& pos,
                             const at::Tensor& freq, const at::Tensor& axes, double amplitude, bool half) {
        const HeadShape s(q);
        const AngleArgs a(pos, freq, axes);
        variable_list out(2);
        int64_t in_s[2][3] = {}, out_s[2][3] = {};
        const at::Tensor* in[2] = {&q, &k};
        for (int i = 0; i < 2; ++i) {
            if (!in[i]->defined()) continue;
            out[i] = empty_like_dtype(in[i]->sizes(), q, q.scalar_type());
            s.strides(*in[i], in_s[i]);
            s.strides(out[i], out_s[i]);
        }
        must(q8k_head_norm(dense_ptr(q), in_s[0], fptr(defined(wq)), out_ptr(out[0]), out_s[0], s.heads(q), dense_ptr(k), in_s[1],
                           fptr(defined(wk)), out_ptr(out[1]), out_s[1], s.heads(k), type_code(q.scalar_type()), (float)eps, a.pos, a.kind, a.stride,
                           a.n_axes, a.axes, a.freq, (float)amplitude, (int)s.batch, (int)s.seq, (int)s.dim, a.rotary_dim, half, stream_of(q)),
             "head_norm");
        return out;
    }
    static variable_list forward(AutogradContext* ctx, const Variable& q, const Maybe& k, const Maybe& wq, const Maybe& wk, double eps,
                                 const Maybe& pos, const Maybe& freq, const Maybe& axes, double amplitude, bool half) {
        variable_list out = run(q, value(k), value(wq), value(wk), eps, value(pos), value(freq), value(axes), amplitude, half);
        ctx->save_for_backward({q, value(k), value(wq), value(wk), value(pos), value(freq), value(axes)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["amplitude"] = amplitude;
        ctx->saved_data["half"] = half;
        ctx->set_materialize_grads(false);
        if (!k.has_value()) out.pop_back();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(10);
        {
            at::NoGradGuard no_grad;
            // the inputs that are there are numbered: q, k, weight of q, weight of k
            const bool there[4] = {true, saved[1].defined(), saved[2].defined(), saved[3].defined()};
            bool need[4];
            for (int i = 0, at = 0; i < 4; ++i) need[i] = there[i] && ctx->needs_input_grad(at++);
            at::Tensor x[2], g[2], dx[2], dw[2], work;
            int64_t xs[2][3] = {}, gs[2][3] = {}, ds[2][3] = {};
            const HeadShape s(saved[0]);
            for (int i = 0; i < 2; ++i) {
                if ((size_t)i >= grads.size() || !grads[i].defined() || !(need[i] || need[2 + i])) continue;
                x[i] = saved[i];
                g[i] = head_grad(grads[i]);
                dx[i] = empty_like_dtype(x[i].sizes(), x[i], x[i].scalar_type());
                if (need[2 + i]) dw[i] = empty_like_dtype({s.dim}, x[i], Dt::Float);
                s.strides(x[i], xs[i]);
                s.strides(g[i], gs[i]);
                s.strides(dx[i], ds[i]);
            }
            if (!x[0].defined() && !x[1].defined()) return result;
            const at::Tensor& some = x[0].defined() ? x[0] : x[1];
            int64_t bytes = 0;
            if (dw[0].defined() || dw[1].defined()) {
                bytes = (int64_t)q8k_head_norm_backward_workspace_bytes((int)s.dim);
                work = empty_like_dtype({bytes}, some, Dt::Byte);
            }
            const AngleArgs a(saved[4], saved[5], saved[6]);
            must_backward(q8k_head_norm_backward(
                              dense_ptr(x[0]), xs[0], fptr(defined(saved[2])), dense_ptr(g[0]), gs[0], out_ptr(dx[0]), ds[0], out_f(dw[0]), s.heads(x[0]),
                              dense_ptr(x[1]), xs[1], fptr(defined(saved[3])), dense_ptr(g[1]), gs[1], out_ptr(dx[1]), ds[1], out_f(dw[1]), s.heads(x[1]),
                              type_code(some.scalar_type()), (float)ctx->saved_data["eps"].toDouble(), a.pos, a.kind, a.stride, a.n_axes, a.axes, a.freq,
                              (float)ctx->saved_data["amplitude"].toDouble(), (int)s.batch, (int)s.seq, (int)s.dim, a.rotary_dim,
                              ctx->saved_data["half"].toBool(), out_ptr(work), (size_t)bytes, stream_of(some)),
                          "head_norm_backward");
            for (int i = 0; i < 2; ++i) {
                if (need[i]) result[i] = dx[i];
                result[2 + i] = dw[i];
            }
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _head_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 10);
    const at::Tensor* q = c.tensor(0, true);
    const at::Tensor* k = c.ok && args[1] != Py_None ? c.tensor(1, true) : nullptr;
    const at::Tensor* wq = c.optional(2, Dt::Float);
    const at::Tensor* wk = c.optional(3, Dt::Float);
    const float eps = c.real(4);
    const at::Tensor* pos = c.ok && args[5] != Py_None ? c.tensor(5, true) : nullptr;
    const at::Tensor* freq = c.ok && args[6] != Py_None ? c.tensor(6) : nullptr;
    const at::Tensor* axes = c.optional(7, Dt::Int);
    const float amplitude = c.real(8);
    const bool half = c.flag(9);
    need_heads(c, q, k, 512);
    need_angles(c, q, pos, freq, axes);
    OR_NONE(c);
    for (const at::Tensor* w : {wq, wk}) c.need(w == nullptr || (w->dim() == 1 && w->size(0) == q->size(-1) && !has_tangent(w)));
    c.need(eps >= 0.f);
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        variable_list out;
        {
            WithoutGil unlocked;
            if (c10::GradMode::is_enabled() && (q->requires_grad() || wants_grad(k) || wants_grad(wq) || wants_grad(wk)))
                out = HeadNormNode::apply(*q, maybe(k), maybe(wq), maybe(wk), (double)eps, maybe(pos), maybe(freq), maybe(axes), (double)amplitude, half);
            else
                out = HeadNormNode::run(*q, value(maybe(k)), value(maybe(wq)), value(maybe(wk)), eps, value(maybe(pos)), value(maybe(freq)),
                                        value(maybe(axes)), amplitude, half);
        }
        return pair_of(std::move(out), k != nullptr);
    });
    FAST_END
}

// ---- _fp4_linear(a, b, bias | None, block scales, row scales | None, gelu, out_type | None): the scales as their types, or their bits (uint8 and
// int32), which is how FP4Linear holds them; row scales are what tells nvfp4 from mxfp4
struct FP4Node : torch::autograd::Function<FP4Node> {
    static at::Tensor run(const at::Tensor& a, const at::Tensor& b, const at::Tensor& bias, const at::Tensor& block, const at::Tensor& row, bool gelu,
                          Dt out_type) {
        const int format = row.defined() ? Q8K_FP4_NV : Q8K_FP4_MX;
        const int64_t k = 2 * b.size(1), nn = b.size(0), m = a.numel() / k;
        at::DimVector shape(lead(a).begin(), lead(a).end());
        shape.push_back(nn);
        at::Tensor out = empty_like_dtype(shape, a, out_type);
        const int64_t bytes = (int64_t)q8k_fp4_linear_workspace_bytes(format, (int)m, (int)nn, (int)k);
        at::Tensor work;
        if (bytes > 0) work = empty_like_dtype({bytes}, a, Dt::Byte);
        must(q8k_fp4_linear(format, a.const_data_ptr(), type_code(a.scalar_type()), b.const_data_ptr(), block.const_data_ptr(),
                            static_cast<const float*>(dense_ptr(row)), fptr(defined(bias)), out.data_ptr(), type_code(out_type), (int)m, (int)nn, (int)k,
                            gelu, out_ptr(work), (size_t)bytes, g_status[a.device().index()]->data_ptr<int>(), stream_of(a)), "fp4_linear");
        return out;
    }
    static Variable forward(AutogradContext* ctx, const Variable& a, const Variable& b, const Maybe& bias, const Variable& block, const Maybe& row,
                            int64_t out_type) {
        Variable out = run(a, b, value(bias), block, value(row), false, (Dt)out_type);
        ctx->save_for_backward({b, block, value(row)});
        ctx->saved_data["type"] = (int64_t)a.scalar_type();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list result(6);
        if (!grads[0].defined()) return result;
        {
            at::NoGradGuard no_grad;
            const at::Tensor &b = saved[0], &block = saved[1], &row = saved[2];
            at::Tensor g = grads[0].contiguous();
            if (reinterpret_cast<uintptr_t>(g.const_data_ptr()) % 16 != 0) g = g.clone();
            const int64_t k = 2 * b.size(1), nn = b.size(0), m = g.numel() / nn;
            at::DimVector shape(lead(g).begin(), lead(g).end());
            shape.push_back(k);
            const Dt type = (Dt)ctx->saved_data["type"].toInt();
            at::Tensor dx = empty_like_dtype(shape, g, type);
            if (m > 0) {
                void* st = stream_of(g);
                auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
                const int64_t work_bytes = up((int64_t)q8k_fp4_weight_operand_workspace_bytes((int)nn, (int)k));
                // one scratch: gradient rows and scales, weight operand and scales, its workspace
                const int64_t at_gs = up(m * nn), at_w = at_gs + up(4 * m), at_ws = at_w + up(k * nn), at_work = at_ws + up(4 * k);
                at::Tensor scratch = empty_like_dtype({at_work + work_bytes}, g, Dt::Byte);
                uint8_t* s = static_cast<uint8_t*>(scratch.data_ptr());
                float *gs = reinterpret_cast<float*>(s + at_gs), *ws = reinterpret_cast<float*>(s + at_ws);
                must_backward(q8k_fp4_backward_quant(g.const_data_ptr(), type_code(g.scalar_type()), s, gs, m, (int)nn, st), "fp4_backward_quant");
                must_backward(q8k_fp4_weight_operand(row.defined() ? Q8K_FP4_NV : Q8K_FP4_MX, b.const_data_ptr(), block.const_data_ptr(),
                                                     static_cast<const float*>(dense_ptr(row)), s + at_w, ws, (int)nn, (int)k, s + at_work,
                                                     (size_t)work_bytes, st), "fp4_weight_operand");
                must_backward(q8k_fp8_mm(s, s + at_w, nullptr, gs, ws, dx.data_ptr(), type_code(type), 1, 1, (int)m, (int)k, (int)nn, 0,
                                         g_status[g.device().index()]->data_ptr<int>(), st), "fp8_mm");
            }
            result[0] = dx;
        }
        return once_only(std::move(result), grads);
    }
};

PyObject* _fp4_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    FAST_BEGIN
    Call c(args, n, 7);
    const at::Tensor* a = c.tensor(0);
    const at::Tensor* b = c.tensor(1, Dt::Byte);
    const at::Tensor* bias = c.optional(2, Dt::Float);
    const at::Tensor* block = c.tensor(3);
    const at::Tensor* row = c.ok && args[4] != Py_None ? c.tensor(4) : nullptr;
    const bool gelu = c.flag(5);
    OR_NONE(c);
    const Dt in = a->scalar_type(), out = c.dtype(6, in);
    auto half_type = [](Dt t) { return t == Dt::BFloat16 || t == Dt::Half; };
    auto aligned = [](const at::Tensor* t) { return reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0; };
    const bool nv = row != nullptr;
    c.need(half_type(in) && half_type(out) && has_rows(a) && b->dim() == 2 && b->size(1) >= 1 && 2 * b->size(1) == a->size(-1) &&
           (block->scalar_type() == Dt::Byte || block->scalar_type() == (nv ? Dt::Float8_e4m3fn : Dt::Float8_e8m0fnu)) &&
           (!nv || row->scalar_type() == Dt::Float || row->scalar_type() == Dt::Int));
    OR_NONE(c);
    const int64_t k = a->size(-1), nn = b->size(0), m = a->numel() / k;
    const bool training = c10::GradMode::is_enabled() && a->requires_grad();
    c.need(aligned(a) && aligned(b) && aligned(block) && k % 32 == 0 && k <= 65536 && nn > 0 && nn % 16 == 0 && nn <= 0x3fffffff && m <= 0x7fffff00 &&
           m * (k / 16) <= 0x7fffffffLL * 128 && block->dim() == 3 && block->size(0) == (nn + 127) / 128 &&
           block->size(1) == (k + 255) / 256 * (nv ? 4 : 2) && block->size(2) == 512 && (!nv || row->numel() == nn) &&
           (bias == nullptr || bias->numel() == nn) && !(training && (gelu || nn > 32768)) && !has_tangent(a) && !has_tangent(bias) && !has_tangent(row));
    c.status();
    OR_NONE(c);
    return answer([&]() -> PyObject* {
        at::Tensor y;
        {
            WithoutGil unlocked;
            y = training ? FP4Node::apply(*a, *b, maybe(bias), *block, maybe(row), (int64_t)out)
                         : FP4Node::run(*a, *b, value(maybe(bias)), *block, value(maybe(row)), gelu, out);
        }
        return wrap(std::move(y));
    });
    FAST_END
}

// ---------------------------------------------------------------- module
PyObject* set_check(PyObject*, PyObject* f) {
    Py_INCREF(f);
    Py_XSETREF(g_check, f);
    Py_RETURN_NONE;
}
// set_status_word(tensor): the word that the launches on its device write when a wait is abandoned
PyObject* set_status_word(PyObject*, PyObject* o) {
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "set_status_word: a tensor is expected");
        return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.scalar_type() != Dt::Int || t.device().index() >= kMaxDevices) {
        PyErr_SetString(PyExc_TypeError, "set_status_word: an int32 CUDA tensor is expected");
        return nullptr;
    }
    at::Tensor*& slot = g_status[t.device().index()];
    if (slot == nullptr) slot = new at::Tensor(t);             // kept for the life of the process, as the device's context is
    else *slot = t;
    Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    FAST(tokenwise_quant), FAST(hadamard_quant), FAST(fast_hadamard_transform), FAST(norm_modulate_quant), FAST(transpose_quant),
    FAST(dequant_hadamard), FAST(rms_norm), FAST(rms_norm_backward), FAST(rope), FAST(rope_backward), FAST(mm),
    FAST(mm_gate_residual), FAST(linear), FAST(flash_attention), FAST(attention_prep_rows), FAST(qk_norm_rope_prep),
    FAST(kv_prep), FAST(qk_norm_rope_prep_pair), FAST(_layer_norm), FAST(_rotary), FAST(_gated_linear),
    FAST(_axial_rotary), FAST(_head_norm), FAST(_fp4_linear),
    {"set_check", set_check, METH_O, nullptr}, {"set_status_word", set_status_word, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "__torch_version__", TORCH_VERSION) != 0) Py_CLEAR(m);
    return m;
}
