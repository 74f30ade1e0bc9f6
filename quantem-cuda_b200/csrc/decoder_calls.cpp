// decoder_calls.cpp — the decoder operators' common calls without the Python
// layers' overhead.
//
// A small product or norm takes a few microseconds on the GPU, and the Python
// checks, allocations and argument lists around it took 9 to 14. These functions
// do the same for the calls that need nothing special: plain contiguous tensors
// of matching shapes and types on the current device. They use tensors through
// Python's object protocol alone (attributes and methods by interned name), so
// the extension stays free of libtorch. Whatever else comes, they return
// NotImplemented and the Python layer checks, converts or raises.
#include "decoder_calls.h"

#include <cstdint>
#include <stdexcept>

#include "quantem_cuda_b200.h"

namespace {

// An owned reference.
class Ref {
public:
    explicit Ref(PyObject *p = nullptr) : p_(p) {}
    ~Ref() { Py_XDECREF(p_); }
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
    Ref(Ref &&o) noexcept : p_(o.p_) { o.p_ = nullptr; }
    Ref &operator=(Ref &&o) noexcept {
        if (this != &o) {
            Py_XDECREF(p_);
            p_ = o.p_;
            o.p_ = nullptr;
        }
        return *this;
    }
    PyObject *get() const { return p_; }
    PyObject *release() {
        PyObject *p = p_;
        p_ = nullptr;
        return p;
    }
    explicit operator bool() const { return p_ != nullptr; }

private:
    PyObject *p_;
};

// A Python exception is set: the call ends with it.
struct Raised {};
// The call is none of the common ones.
struct Uncommon {};

struct Names {
    PyObject *shape, *dtype, *data_ptr, *is_contiguous, *get_device, *new_empty, *requires_grad;
    PyObject *kw_dtype;  // ("dtype",)
} names;

constexpr int kTypes = 4;
// What setup() was given, kept for the life of the process.
PyObject *tensor_type, *parameter_type, *dtypes[kTypes], *uint8_dtype, *current_device, *current_stream, *grad_enabled,
    *activations, *dispatch_modes, *function_modes, *forward_ad, *forward_ad_level;

PyObject *checked(PyObject *p) {
    if (!p) throw Raised();
    return p;
}
void require(bool common) {
    if (!common) throw Uncommon();
}

long long as_int(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}
long long call_int(PyObject *self, PyObject *name) {
    PyObject *args[1] = {self};
    Ref r(checked(PyObject_VectorcallMethod(name, args, 1, nullptr)));
    return as_int(r.get());
}

constexpr int kMaxDims = 8;

// A plain contiguous CUDA tensor.
struct Arg {
    PyObject *o = nullptr;
    int type = -1, dims = 0;
    long long size[kMaxDims], count = 1;
    long long device = -1;
    uintptr_t ptr = 0;

    // `o` may be None: then `ptr` stays 0
    Arg(PyObject *obj, bool may_lack) {
        if (obj == Py_None) {
            require(may_lack);
            return;
        }
        require((PyObject *)Py_TYPE(obj) == tensor_type || (PyObject *)Py_TYPE(obj) == parameter_type);
        o = obj;
        Ref t(checked(PyObject_GetAttr(o, names.dtype)));
        for (int i = 0; i < kTypes; ++i)
            if (t.get() == dtypes[i]) type = i;
        require(type >= 0);
        PyObject *args[1] = {o};
        Ref c(checked(PyObject_VectorcallMethod(names.is_contiguous, args, 1, nullptr)));
        require(c.get() == Py_True);
        device = call_int(o, names.get_device);
        require(device >= 0);
        Ref s(checked(PyObject_GetAttr(o, names.shape)));
        require(PyTuple_Check(s.get()) && PyTuple_GET_SIZE(s.get()) <= kMaxDims);
        dims = (int)PyTuple_GET_SIZE(s.get());
        for (int i = 0; i < dims; ++i) {
            PyObject *v = PyTuple_GET_ITEM(s.get(), i);
            require(PyLong_CheckExact(v));  // torch.jit.trace gives tensors
            size[i] = as_int(v);
            count *= size[i];
        }
        ptr = (uintptr_t)call_int(o, names.data_ptr);
        require(ptr != 0 || count == 0);  // torch.func's tensors have no address of their own
    }
    bool given() const { return o != nullptr; }
    long long last() const { return size[dims - 1]; }
    bool alike(const Arg &b) const {  // same shape and device
        if (dims != b.dims || device != b.device) return false;
        for (int i = 0; i < dims; ++i)
            if (size[i] != b.size[i]) return false;
        return true;
    }
    bool vector(long long n, const Arg &on) const { return dims == 1 && size[0] == n && device == on.device; }
    // shape of `b` with the last dimension replaced by n (n < 0: left out)
    bool rows_of(const Arg &b, long long n) const {
        if (dims != b.dims - (n < 0) || device != b.device) return false;
        for (int i = 0; i < b.dims - 1; ++i)
            if (size[i] != b.size[i]) return false;
        return n < 0 || last() == n;
    }
};

// A call that comes straight from a user: none that a mode records (make_fx has
// a function mode where it has no dispatch mode) and none inside a forward-mode
// level, whose tangents the outputs' allocations would drop.
void require_direct() {
    Ref level(checked(PyObject_GetAttr(forward_ad, forward_ad_level)));
    require(as_int(level.get()) < 0);
    Ref d(checked(PyObject_CallNoArgs(dispatch_modes)));
    require(as_int(d.get()) == 0);
    Ref f(checked(PyObject_CallNoArgs(function_modes)));
    require(as_int(f.get()) == 0);
}

// Whether a gradient is recorded for one of the plain tensors (or None) in
// a[0..n); asked before anything else, as the answer sends the call on.
bool wants_grad(PyObject *const *a, int n) {
    Ref on(checked(PyObject_CallNoArgs(grad_enabled)));
    if (on.get() != Py_True) return false;
    bool wants = false;
    for (int i = 0; i < n; ++i) {
        if (a[i] == Py_None) continue;
        require((PyObject *)Py_TYPE(a[i]) == tensor_type || (PyObject *)Py_TYPE(a[i]) == parameter_type);
        Ref r(checked(PyObject_GetAttr(a[i], names.requires_grad)));
        wants = wants || r.get() == Py_True;
    }
    return wants;
}

// The current stream, if x's device is the current one.
cudaStream_t stream_on(const Arg &x) {
    Ref d(checked(PyObject_CallNoArgs(current_device)));
    require(as_int(d.get()) == x.device);
    Ref s(checked(PyObject_CallOneArg(current_stream, d.get())));
    return reinterpret_cast<cudaStream_t>((uintptr_t)as_int(s.get()));
}

Ref new_tensor(const Arg &like, PyObject *shape, PyObject *dtype) {
    PyObject *args[3] = {like.o, shape, dtype};
    return Ref(checked(PyObject_VectorcallMethod(names.new_empty, args, 2, dtype ? names.kw_dtype : nullptr)));
}
// like.shape with the last dimension replaced by n (n < 0: left out)
Ref shape_of(const Arg &like, long long n) {
    const int dims = like.dims - (n < 0);
    Ref s(checked(PyTuple_New(dims)));
    for (int i = 0; i < dims; ++i)
        PyTuple_SET_ITEM(s.get(), i, checked(PyLong_FromLongLong(i == like.dims - 1 ? n : like.size[i])));
    return s;
}
uintptr_t address(const Ref &t) { return (uintptr_t)call_int(t.get(), names.data_ptr); }

Ref bytes_like(const Arg &like, size_t bytes) {
    Ref n(checked(PyLong_FromSize_t(bytes)));
    return new_tensor(like, n.get(), uint8_dtype);
}

template <typename T>
T *ptr(uintptr_t v) {
    return reinterpret_cast<T *>(v);
}

void check(int status) {
    if (status == 0) return;
    PyErr_Format(PyExc_RuntimeError, "%s: %s", quantem_cuda_status_string(status), quantem_cuda_last_error());
    throw Raised();
}

int activation_of(PyObject *name) {
    require(PyUnicode_Check(name));
    PyObject *code = PyDict_GetItemWithError(activations, name);
    if (!code && PyErr_Occurred()) throw Raised();
    require(code != nullptr);
    return (int)as_int(code);
}
int type_of(PyObject *dtype, int standard) {
    if (dtype == Py_None) return standard;
    for (int i = 0; i < kTypes; ++i)
        if (dtype == dtypes[i]) return i;
    throw Uncommon();
}
bool is_16bit(int t) { return t == QC_BF16 || t == QC_F16; }

template <typename F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F &&body) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd given", want, got);
        return nullptr;
    }
    try {
        return body();
    } catch (const Raised &) {
        return nullptr;
    } catch (const Uncommon &) {
        Py_RETURN_NOTIMPLEMENTED;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype, from_user) -> y,
// or None where a user's tensors are plain and a gradient is recorded
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 9, [&]() -> PyObject * {
        if (a[8] == Py_True) {
            require_direct();
            if (wants_grad(a, 6)) Py_RETURN_NONE;
        }
        const Arg x(a[0], false), w(a[1], false), b(a[2], true), r(a[3], true), sx(a[4], true), sw(a[5], true);
        const bool f8 = sx.given();
        require(x.type == w.type && (f8 ? x.type == QC_E4M3 : is_16bit(x.type)) && x.dims >= 1 && w.dims == 2);
        const long long k = x.last(), n = w.size[0];
        require(k > 0 && n > 0 && w.size[1] == k && w.device == x.device && k < (1 << 30) && n < (1 << 30));
        const int out = type_of(a[7], f8 ? QC_BF16 : x.type);
        require(out == QC_F32 || (f8 ? is_16bit(out) : out == x.type));
        if (b.given()) require(b.vector(n, x) && (b.type == QC_F32 || (f8 ? is_16bit(b.type) : b.type == x.type)));
        if (r.given()) require(r.type == out && r.rows_of(x, n));
        if (f8) require(sw.given() && sx.type == QC_F32 && sw.type == QC_F32 && sx.rows_of(x, -1) && sw.vector(n, x));
        else require(!sw.given());
        const int act = activation_of(a[6]);
        const cudaStream_t stream = stream_on(x);
        Ref y = new_tensor(x, shape_of(x, n).get(), out == x.type ? nullptr : dtypes[out]), ws;
        const long rows = (long)(x.count / k);
        const size_t bytes = linear_act_workspace_bytes(ptr<const void>(x.ptr), ptr<const void>(w.ptr), rows, (int)n,
                                                        (int)k, (long)k, (long)k, x.type);
        if (bytes) ws = bytes_like(x, bytes);
        check(linear_act_cuda(ptr<const void>(x.ptr), ptr<const void>(w.ptr), ptr<const void>(b.ptr),
                              ptr<const void>(r.ptr), ptr<void>(address(y)), ptr<const float>(sx.ptr),
                              ptr<const float>(sw.ptr), rows, (int)n, (int)k, (long)k, (long)k, (long)n, x.type, out,
                              b.given() ? b.type : 0, act, ws ? ptr<void>(address(ws)) : nullptr, bytes, stream));
        return y.release();
    });
}

// (x, weight, bias, residual, activation, out_dtype) -> (y, kept), or
// NotImplemented where the call keeps nothing for its backward
PyObject *linear_keep(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 6, [&]() -> PyObject * {
        const Arg x(a[0], false);
        if (x.type != QC_BF16 || x.dims < 1) Py_RETURN_NOTIMPLEMENTED;
        const Arg w(a[1], false), b(a[2], true), r(a[3], true);
        require(w.type == x.type && w.dims == 2);
        const long long k = x.last(), n = w.size[0];
        require(k > 0 && n > 0 && w.size[1] == k && w.device == x.device && k < (1 << 30) && n < (1 << 30));
        const int act = activation_of(a[4]);
        const long rows = (long)(x.count / k);
        const size_t kept_bytes = linear_act_kept_bytes(rows, (int)n, (int)k, x.type, type_of(a[5], x.type),
                                                        b.given() ? b.type : QC_BF16, act);
        if (!kept_bytes) Py_RETURN_NOTIMPLEMENTED;
        if (b.given()) require(b.vector(n, x) && b.type == x.type);
        if (r.given()) require(r.type == x.type && r.rows_of(x, n));
        const cudaStream_t stream = stream_on(x);
        Ref y = new_tensor(x, shape_of(x, n).get(), nullptr), kept = bytes_like(x, kept_bytes), ws;
        const size_t bytes = linear_act_workspace_bytes(ptr<const void>(x.ptr), ptr<const void>(w.ptr), rows, (int)n,
                                                        (int)k, (long)k, (long)k, x.type);
        if (bytes) ws = bytes_like(x, bytes);
        check(linear_act_keep_cuda(ptr<const void>(x.ptr), ptr<const void>(w.ptr), ptr<const void>(b.ptr),
                                   ptr<const void>(r.ptr), ptr<void>(address(y)), ptr<void>(address(kept)), rows, (int)n,
                                   (int)k, (long)k, (long)k, (long)n, x.type, x.type, act,
                                   ws ? ptr<void>(address(ws)) : nullptr, bytes, stream));
        return PyTuple_Pack(2, y.get(), kept.get());
    });
}

// (x, weight, kept, dy, activation, need_dx, need_dweight, need_dbias) -> (dx, dweight, dbias)
PyObject *linear_grad_kept(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 8, [&]() -> PyObject * {
        const Arg x(a[0], false), w(a[1], false), dy(a[3], false);
        require(x.type == QC_BF16 && w.type == x.type && x.dims >= 1 && w.dims == 2);
        const long long k = x.last(), n = w.size[0];
        require(k > 0 && w.size[1] == k && w.device == x.device);
        require(dy.type == x.type && dy.rows_of(x, n) && dy.ptr % 16 == 0);
        const int act = activation_of(a[4]);
        const cudaStream_t stream = stream_on(x);
        Ref dx, dw, db, ws;
        if (a[5] == Py_True) dx = new_tensor(x, shape_of(x, k).get(), nullptr);
        if (a[6] == Py_True) dw = new_tensor(w, shape_of(w, k).get(), nullptr);
        if (a[7] == Py_True) {
            Ref shape(checked(PyTuple_Pack(1, Ref(checked(PyLong_FromLongLong(n))).get())));
            db = new_tensor(x, shape.get(), nullptr);
        }
        void *pdx = dx ? ptr<void>(address(dx)) : nullptr, *pdw = dw ? ptr<void>(address(dw)) : nullptr,
             *pdb = db ? ptr<void>(address(db)) : nullptr;
        const long rows = (long)(x.count / k);
        const void *px = ptr<const void>(x.ptr), *pw = ptr<const void>(w.ptr), *pdy = ptr<const void>(dy.ptr);
        const size_t bytes = linear_act_grad_kept_workspace_bytes(px, pw, pdy, pdx, pdw, pdb, rows, (int)n, (int)k,
                                                                  (long)k, (long)k, (long)n, x.type, act, (int)x.device);
        if (bytes) ws = bytes_like(x, bytes);
        check(linear_act_grad_kept_cuda(px, pw, ptr<const void>((uintptr_t)call_int(a[2], names.data_ptr)), pdy, pdx,
                                        pdw, pdb, rows, (int)n, (int)k, (long)k, (long)k, (long)n, x.type, act,
                                        ws ? ptr<void>(address(ws)) : nullptr, bytes, stream));
        return PyTuple_Pack(3, dx ? dx.get() : Py_None, dw ? dw.get() : Py_None, db ? db.get() : Py_None);
    });
}

// (x, weight, bias, dy, activation, need_dx, need_dweight, need_dbias) -> (dx, dweight, dbias)
PyObject *linear_grad(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 8, [&]() -> PyObject * {
        const Arg x(a[0], false), w(a[1], false), b(a[2], true), dy(a[3], false);
        require(x.type == w.type && is_16bit(x.type) && x.dims >= 1 && w.dims == 2);
        const long long k = x.last(), n = w.size[0];
        require(k > 0 && n > 0 && w.size[1] == k && w.device == x.device && k < (1 << 30) && n < (1 << 30));
        require((dy.type == x.type || dy.type == QC_F32) && dy.rows_of(x, n));
        if (b.given()) require(b.vector(n, x) && (b.type == QC_F32 || b.type == x.type));
        const int act = activation_of(a[4]);
        const cudaStream_t stream = stream_on(x);
        Ref dx, dw, db, ws;
        if (a[5] == Py_True) dx = new_tensor(x, shape_of(x, k).get(), nullptr);
        if (a[6] == Py_True) dw = new_tensor(w, shape_of(w, k).get(), nullptr);
        if (a[7] == Py_True && b.given()) db = new_tensor(b, shape_of(b, n).get(), nullptr);
        void *pdx = dx ? ptr<void>(address(dx)) : nullptr, *pdw = dw ? ptr<void>(address(dw)) : nullptr,
             *pdb = db ? ptr<void>(address(db)) : nullptr;
        const long rows = (long)(x.count / k);
        const void *px = ptr<const void>(x.ptr), *pw = ptr<const void>(w.ptr), *pdy = ptr<const void>(dy.ptr);
        const size_t bytes = linear_act_grad_workspace_bytes(px, pw, pdy, pdx, pdw, pdb, rows, (int)n, (int)k, (long)k,
                                                             (long)k, (long)n, x.type, dy.type, act, (int)x.device);
        if (bytes) ws = bytes_like(x, bytes);
        check(linear_act_grad_cuda(px, pw, ptr<const void>(b.ptr), pdy, pdx, pdw, pdb, rows, (int)n, (int)k, (long)k,
                                   (long)k, (long)n, x.type, dy.type, b.given() ? b.type : 0, act,
                                   ws ? ptr<void>(address(ws)) : nullptr, bytes, stream));
        return PyTuple_Pack(3, dx ? dx.get() : Py_None, dw ? dw.get() : Py_None, db ? db.get() : Py_None);
    });
}

// (x, residual, weight, eps, out_dtype, from_user) -> (y[, scale][, h]), the
// scale for out_dtype e4m3; None as above
PyObject *norm(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 6, [&]() -> PyObject * {
        if (a[5] == Py_True) {
            require_direct();
            if (wants_grad(a, 3)) Py_RETURN_NONE;
        }
        const Arg x(a[0], false), r(a[1], true), w(a[2], false);
        require(x.type != QC_E4M3 && x.dims >= 1 && x.last() > 0 && x.last() < (1 << 30));
        const long long n = x.last();
        const int out = type_of(a[4], x.type);
        require(w.type == x.type && w.vector(n, x));
        if (r.given()) require(r.type == x.type && r.alike(x));
        require(PyFloat_CheckExact(a[3]));
        require(out == x.type || out == QC_F32 || out == QC_E4M3 || x.type == QC_F32);
        const cudaStream_t stream = stream_on(x);
        Ref shape = shape_of(x, n), scale, h;
        Ref y = new_tensor(x, shape.get(), out == x.type ? nullptr : dtypes[out]);
        if (out == QC_E4M3)
            scale = new_tensor(x, shape_of(x, -1).get(), x.type == QC_F32 ? nullptr : dtypes[QC_F32]);
        if (r.given()) h = new_tensor(x, shape.get(), nullptr);
        const void *px = ptr<const void>(x.ptr);
        const long rows = (long)(x.count / n);
        float *ps = scale ? ptr<float>(address(scale)) : nullptr;
        check(rms_norm_cuda(px, ptr<const void>(r.ptr), ptr<const void>(w.ptr), ptr<void>(address(y)),
                            h ? ptr<void>(address(h)) : nullptr, ps, rows, (int)n, (long)n, (long)n, x.type, out,
                            (float)PyFloat_AS_DOUBLE(a[3]), stream));
        if (scale && h) return PyTuple_Pack(3, y.get(), scale.get(), h.get());
        if (scale || h) return PyTuple_Pack(2, y.get(), scale ? scale.get() : h.get());
        return PyTuple_Pack(1, y.get());
    });
}

// (x, from_user) -> (q, scale); None as above
PyObject *quantize(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 2, [&]() -> PyObject * {
        if (a[1] == Py_True) {
            require_direct();
            if (wants_grad(a, 1)) Py_RETURN_NONE;
        }
        const Arg x(a[0], false);
        require(x.type != QC_E4M3 && x.dims >= 1 && x.last() > 0 && x.last() < (1 << 30));
        const long long n = x.last();
        const cudaStream_t stream = stream_on(x);
        Ref q = new_tensor(x, shape_of(x, n).get(), dtypes[QC_E4M3]);
        Ref scale = new_tensor(x, shape_of(x, -1).get(), x.type == QC_F32 ? nullptr : dtypes[QC_F32]);
        check(quantize_rows_cuda(ptr<const void>(x.ptr), ptr<void>(address(q)), ptr<float>(address(scale)),
                                 (long)(x.count / n), (int)n, (long)n, x.type, stream));
        return PyTuple_Pack(2, q.get(), scale.get());
    });
}

// (x, residual, weight, dy, dh, eps, need_dx, need_dweight) -> (dx, dweight)
PyObject *norm_grad(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 8, [&]() -> PyObject * {
        const Arg x(a[0], false), r(a[1], true), w(a[2], false), dy(a[3], false), dh(a[4], true);
        require(x.type != QC_E4M3 && x.dims >= 1 && x.last() > 0 && x.last() < (1 << 30));
        const long long n = x.last();
        require(w.type == x.type && w.vector(n, x));
        if (r.given()) require(r.type == x.type && r.alike(x));
        require(dy.alike(x) && (dy.type == x.type || dy.type == QC_F32 || (x.type == QC_F32 && is_16bit(dy.type))));
        if (dh.given()) require(dh.type == x.type && dh.alike(x));
        require(PyFloat_CheckExact(a[5]));
        const cudaStream_t stream = stream_on(x);
        Ref dx, dw, ws;
        if (a[6] == Py_True) dx = new_tensor(x, shape_of(x, n).get(), nullptr);
        if (a[7] == Py_True) dw = new_tensor(w, shape_of(w, n).get(), nullptr);
        const long rows = (long)(x.count / n);
        const size_t bytes = dw ? rms_norm_grad_workspace_bytes(rows, (int)n) : 0;
        if (bytes) ws = bytes_like(x, bytes);
        check(rms_norm_grad_cuda(ptr<const void>(x.ptr), ptr<const void>(r.ptr), ptr<const void>(w.ptr),
                                 ptr<const void>(dy.ptr), ptr<const void>(dh.ptr),
                                 dx ? ptr<void>(address(dx)) : nullptr, dw ? ptr<void>(address(dw)) : nullptr, rows,
                                 (int)n, (long)n, (long)n, (long)n, (long)n, x.type, dy.type,
                                 (float)PyFloat_AS_DOUBLE(a[5]), ws ? ptr<void>(address(ws)) : nullptr, bytes, stream));
        return PyTuple_Pack(2, dx ? dx.get() : Py_None, dw ? dw.get() : Py_None);
    });
}

// (Tensor, Parameter, (dtypes in the order of QC_F32..QC_E4M3), uint8, current
// device's index, raw current stream, is_grad_enabled, {activation: code},
// dispatch modes' and function modes' number, torch.autograd.forward_ad)
PyObject *setup(PyObject *, PyObject *const *a, Py_ssize_t n_args) {
    return guarded(n_args, 11, [&]() -> PyObject * {
        require(PyTuple_Check(a[2]) && PyTuple_GET_SIZE(a[2]) == kTypes && PyDict_Check(a[7]));
        const char *words[] = {"shape", "dtype", "data_ptr", "is_contiguous", "get_device", "new_empty", "requires_grad"};
        PyObject **to[] = {&names.shape,      &names.dtype,     &names.data_ptr,     &names.is_contiguous,
                           &names.get_device, &names.new_empty, &names.requires_grad};
        for (int i = 0; i < 7; ++i) *to[i] = checked(PyUnicode_InternFromString(words[i]));
        names.kw_dtype = checked(PyTuple_Pack(1, names.dtype));
        tensor_type = Py_NewRef(a[0]);
        parameter_type = Py_NewRef(a[1]);
        for (int i = 0; i < kTypes; ++i) dtypes[i] = Py_NewRef(PyTuple_GET_ITEM(a[2], i));
        uint8_dtype = Py_NewRef(a[3]);
        current_device = Py_NewRef(a[4]);
        current_stream = Py_NewRef(a[5]);
        grad_enabled = Py_NewRef(a[6]);
        activations = Py_NewRef(a[7]);
        dispatch_modes = Py_NewRef(a[8]);
        function_modes = Py_NewRef(a[9]);
        forward_ad = Py_NewRef(a[10]);
        forward_ad_level = checked(PyUnicode_InternFromString("_current_level"));
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    {"decoder_setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, "Types and functions the calls below use."},
    {"decoder_linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL,
     "linear_act / linear_act_fp8 for plain contiguous tensors, or NotImplemented."},
    {"decoder_linear_grad", (PyCFunction)(void (*)(void))linear_grad, METH_FASTCALL,
     "Backward of linear_act for plain contiguous tensors, or NotImplemented."},
    {"decoder_linear_keep", (PyCFunction)(void (*)(void))linear_keep, METH_FASTCALL,
     "linear_act with the activation's derivative kept for the backward, or NotImplemented."},
    {"decoder_linear_grad_kept", (PyCFunction)(void (*)(void))linear_grad_kept, METH_FASTCALL,
     "Backward of linear_act from the kept derivative, or NotImplemented."},
    {"decoder_norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL,
     "RMS norm for plain contiguous tensors, or NotImplemented."},
    {"decoder_quantize", (PyCFunction)(void (*)(void))quantize, METH_FASTCALL,
     "quantize_rows_fp8 for plain contiguous tensors, or NotImplemented."},
    {"decoder_norm_grad", (PyCFunction)(void (*)(void))norm_grad, METH_FASTCALL,
     "Backward of the RMS norm for plain contiguous tensors, or NotImplemented."},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

int add_decoder_calls(PyObject *module) { return PyModule_AddFunctions(module, methods); }
