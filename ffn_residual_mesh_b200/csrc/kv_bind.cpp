// Python binding of the paged cache's calls: argument checks and the C ABI call in one step, so that a
// call costs about as much as its launch. Functions take positional arguments from
// ffn_residual_mesh_b200/kvcache.py; `geo` is (handle, kv_heads, head_dim, device index).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/StreamGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <exception>
#include <initializer_list>

#include "ffnrm.h"

namespace {

// An error that is already set, or a message for ValueError.
struct Refused : std::exception {};
[[noreturn]] void refuse(const char *fmt, ...) {
    char buf[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    PyErr_SetString(PyExc_ValueError, buf);
    throw Refused();
}

void check(int rc) {
    if (rc == FFNRM_OK) return;
    const char *msg = ffnrm_last_error();
    if (rc == FFNRM_ERR_ARG)
        PyErr_SetString(PyExc_ValueError, msg);
    else if (rc == FFNRM_ERR_NOMEM)
        PyErr_SetString(PyExc_MemoryError, msg);
    else if (rc == FFNRM_ERR_TIMEOUT)
        PyErr_SetString(PyExc_TimeoutError, msg);
    else
        PyErr_Format(PyExc_RuntimeError, "ffnrm error %d: %s", rc, msg);
    throw Refused();
}

const at::Tensor &tensor(const char *name, PyObject *o) {
    if (!THPVariable_Check(o)) refuse("%s must be a torch tensor, got %s", name, Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    return v;
}

int int32_of(const char *name, int64_t v) {
    if (v < INT32_MIN || v > INT32_MAX) refuse("%s=%lld does not fit 32 bits", name, (long long)v);
    return int(v);
}

struct Geo {
    ffnrm_kv *kv;
    int64_t heads, dim;
    int device;
    explicit Geo(PyObject *t) {
        if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 4) refuse("the cache is closed");
        kv = reinterpret_cast<ffnrm_kv *>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(t, 0)));
        heads = integer(PyTuple_GET_ITEM(t, 1));
        dim = integer(PyTuple_GET_ITEM(t, 2));
        device = int(integer(PyTuple_GET_ITEM(t, 3)));
        if (!kv) refuse("the cache is closed");
    }
};

void on(const char *name, const at::Tensor &x, int device) {
    if (!x.is_cuda() || x.get_device() != device)
        refuse("%s must be on cuda:%d, got %s", name, device, x.device().str().c_str());
}

int dtype_of(const at::Tensor &x) {
    switch (x.scalar_type()) {
        case at::kHalf: return FFNRM_F16;
        case at::kBFloat16: return FFNRM_BF16;
        case at::kFloat: return FFNRM_F32;
        default: refuse("expected float16, bfloat16 or float32, got %s", at::toString(x.scalar_type()));
    }
}

// A [rows, heads, dim] view with contiguous channels; rows < 0: any number.
ffnrm_rows rows_of(const char *name, const at::Tensor &x, int64_t rows, int64_t heads, int64_t dim, int device) {
    if (x.dim() != 3 || x.size(1) != heads || x.size(2) != dim || (rows >= 0 && x.size(0) != rows))
        refuse("%s must have shape (%lld, %lld, %lld) (-1: any), got %zu dimensions of %lld x %lld x %lld", name, (long long)rows,
               (long long)heads, (long long)dim, size_t(x.dim()), (long long)(x.dim() > 0 ? x.size(0) : 0),
               (long long)(x.dim() > 1 ? x.size(1) : 0), (long long)(x.dim() > 2 ? x.size(2) : 0));
    if (x.stride(2) != 1 && dim > 1 && x.numel()) refuse("%s must have contiguous channels", name);
    on(name, x, device);
    return ffnrm_rows{x.data_ptr(), x.stride(0), x.stride(1)};
}

// A tensor that is written must not name one element twice (an expanded view).
void writable(const char *name, const at::Tensor &x) {
    for (int64_t i = 0; i < x.dim(); ++i)
        if (x.stride(i) == 0 && x.size(i) > 1) refuse("%s must not be an expanded view", name);
}

// A caller's tensor has new contents: autograd's saved copies of it are out of date.
void written(PyObject *o) {
    if (o == Py_None) return;
    const at::Tensor &x = THPVariable_Unpack(o);
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

int32_t *ints(const char *name, const at::Tensor &x, int device) {
    if (x.scalar_type() != at::kInt || !x.is_contiguous()) refuse("%s must be a contiguous int32 tensor", name);
    on(name, x, device);
    return x.data_ptr<int32_t>();
}
int32_t *ints1(const char *name, const at::Tensor &x, int64_t n, int device) {
    if (x.dim() != 1 || x.size(0) != n) refuse("%s must have shape (%lld,)", name, (long long)n);
    return ints(name, x, device);
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int device) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, c10::DeviceIndex(device)));
}

// The call's stream: the current one, or the one that is given, which is then current for the call, so
// that a new output's memory belongs to the stream that writes it. `keep` holds the caller's tensors, which
// belong to other streams, until the call's work on it is done, should the caller drop them before.
struct Stream {
    c10::OptionalStreamGuard guard;
    void *ptr;
    bool other = false;  // not the current stream
    void keep(std::initializer_list<PyObject *> tensors) const {
        if (!other) return;
        const c10::Stream stream = *guard.current_stream();
        for (PyObject *o : tensors)
            if (THPVariable_Check(o)) THPVariable_Unpack(o).record_stream(stream);
    }
    Stream(PyObject *o, int device) {
        const c10::DeviceIndex d(device);
        if (o == Py_None) {
            ptr = c10::cuda::getCurrentCUDAStream(d).stream();
            return;
        }
        if (PyLong_Check(o)) {
            ptr = PyLong_AsVoidPtr(o);
        } else {
            PyObject *v = PyObject_GetAttrString(o, "cuda_stream");
            if (!v) throw Refused();
            ptr = PyLong_AsVoidPtr(v);
            Py_DECREF(v);
        }
        if (!ptr && PyErr_Occurred()) throw Refused();
        other = ptr != c10::cuda::getCurrentCUDAStream(d).stream();
        guard.reset_stream(ptr ? c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(ptr), d)
                               : c10::cuda::getDefaultCUDAStream(d));
    }
};

ffnrm_kv_batch batch_of(PyObject *tables, PyObject *lengths, PyObject *starts, int64_t rows, int device) {
    const at::Tensor &t = tensor("tables", tables);
    if (t.dim() != 2) refuse("tables must have shape (seqs, width)");
    ffnrm_kv_batch b{};
    b.seqs = int32_of("seqs", t.size(0));
    b.table_width = int32_of("table width", t.size(1));
    b.rows = int32_of("rows", rows);
    b.tables = ints("tables", t, device);
    b.lengths = ints1("lengths", tensor("lengths", lengths), t.size(0), device);
    if (starts != Py_None) b.starts = ints1("starts", tensor("starts", starts), t.size(0) + 1, device);
    return b;
}

template <PyObject *(*F)(PyObject *const *)>
PyObject *guarded(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
        return nullptr;
    }
}

// x, positions, cos_sin, out or None, flags, stream. None (and nothing done) for an x that autograd follows.
PyObject *rotary(PyObject *const *a) {
    const at::Tensor &x = tensor("x", a[0]), &table = tensor("table", a[2]);
    if (x.dim() != 3) refuse("x must have shape (T, heads, dim)");
    if (!x.is_cuda()) refuse("x must be on a CUDA device");
    if (at::GradMode::is_enabled() && (x.requires_grad() || (a[3] != Py_None && tensor("out", a[3]).requires_grad()))) {
        if (a[3] != Py_None) refuse("out= takes no part in autograd: x and out must not require a gradient");
        Py_RETURN_NONE;
    }
    const int device = x.get_device(), dtype = dtype_of(x);
    const Stream stream(a[5], device);
    const int64_t T = x.size(0), heads = x.size(1), dim = x.size(2);
    if (table.size(1) > dim) refuse("rotary_dim=%lld exceeds head dim %lld", (long long)table.size(1), (long long)dim);
    on("table", table, device);
    at::Tensor out;
    if (a[3] == Py_None) {
        out = empty({T, heads, dim}, x.scalar_type(), device);
    } else {
        out = tensor("out", a[3]);
        if (out.scalar_type() != x.scalar_type()) refuse("out must have x's type");
        writable("out", out);
    }
    const ffnrm_rows xr = rows_of("x", x, T, heads, dim, device), yr = rows_of("out", out, T, heads, dim, device);
    const int32_t *pos = ints1("positions", tensor("positions", a[1]), T, device);
    const c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
    check(ffnrm_rotary(&xr, &yr, dtype, int32_of("T", T), int32_of("heads", heads), int32_of("dim", dim), pos, table.data_ptr<float>(),
                       int32_of("rotary_dim", table.size(1)), int32_of("max_positions", table.size(0)), int(integer(a[4])),
                       stream.ptr));
    stream.keep({a[0], a[1], a[2], a[3]});
    written(a[3]);
    return THPVariable_Wrap(std::move(out));
}

// geo, layer, k, v, tables, lengths, starts, cos_sin or None, flags, q or None, q_out or None, stream
PyObject *append(PyObject *const *a) {
    const Geo geo(a[0]);
    const Stream stream(a[11], geo.device);
    const at::Tensor &k = tensor("k", a[2]), &v = tensor("v", a[3]);
    const ffnrm_rows kr = rows_of("k", k, -1, geo.heads, geo.dim, geo.device);
    const int64_t T = k.size(0);
    const ffnrm_rows vr = rows_of("v", v, T, geo.heads, geo.dim, geo.device);
    const int dtype = dtype_of(k);
    if (v.scalar_type() != k.scalar_type()) refuse("q, k and v must have one type");
    const ffnrm_kv_batch batch = batch_of(a[4], a[5], a[6], T, geo.device);
    const float *table = nullptr;
    int rot = 0, positions = 0;
    if (a[7] != Py_None) {
        const at::Tensor &t = tensor("rope", a[7]);
        on("rope", t, geo.device);
        table = t.data_ptr<float>();
        rot = int32_of("rotary_dim", t.size(1));
        positions = int32_of("max_positions", t.size(0));
    }
    ffnrm_rows qr{}, yr{};
    at::Tensor out;
    int64_t heads = 0;
    if (a[9] != Py_None) {
        const at::Tensor &q = tensor("q", a[9]);
        if (!table) refuse("q is only rotated: it needs rope");
        if (q.scalar_type() != k.scalar_type()) refuse("q, k and v must have one type");
        heads = q.dim() == 3 ? q.size(1) : -1;
        qr = rows_of("q", q, T, heads, geo.dim, geo.device);
        if (a[10] == Py_None) {
            out = empty({T, heads, geo.dim}, q.scalar_type(), geo.device);
        } else {
            out = tensor("q_out", a[10]);
            if (out.scalar_type() != q.scalar_type()) refuse("q_out must have q's type");
            writable("q_out", out);
        }
        yr = rows_of("q_out", out, T, heads, geo.dim, geo.device);
        if (T == 0) qr.data = yr.data = nullptr;
    }
    const int layer = int32_of("layer", integer(a[1]));
    check(ffnrm_kv_append(geo.kv, layer, &batch, dtype, &kr, &vr, &qr, &yr, int32_of("heads", heads), table, rot, positions,
                          int(integer(a[8])), stream.ptr));
    stream.keep({a[2], a[3], a[4], a[5], a[6], a[7], a[9], a[10]});
    if (!out.defined()) Py_RETURN_NONE;
    written(a[10]);
    return THPVariable_Wrap(std::move(out));
}

// geo, layer, q, tables, lengths, starts, out or None, lse or None, scale, causal, window, stream
PyObject *attend(PyObject *const *a) {
    const Geo geo(a[0]);
    const Stream stream(a[11], geo.device);
    const at::Tensor &q = tensor("q", a[2]);
    if (q.dim() != 3 || q.size(1) == 0 || q.size(1) % geo.heads)
        refuse("q must have shape (T, a multiple of %lld, %lld)", (long long)geo.heads, (long long)geo.dim);
    const int64_t T = q.size(0), heads = q.size(1);
    const int dtype = dtype_of(q);
    const ffnrm_rows qr = rows_of("q", q, T, heads, geo.dim, geo.device);
    const ffnrm_kv_batch batch = batch_of(a[3], a[4], a[5], T, geo.device);
    at::Tensor out;
    if (a[6] == Py_None) {
        out = empty({T, heads, geo.dim}, q.scalar_type(), geo.device);
    } else {
        out = tensor("out", a[6]);
        if (out.scalar_type() != q.scalar_type()) refuse("out must have q's type");
        writable("out", out);
    }
    const ffnrm_rows yr = rows_of("out", out, T, heads, geo.dim, geo.device);
    float *lse = nullptr;
    if (a[7] != Py_None) {
        const at::Tensor &t = tensor("lse", a[7]);
        if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != T || t.size(1) != heads || !t.is_contiguous())
            refuse("lse must be a contiguous float32 tensor of shape (%lld, %lld)", (long long)T, (long long)heads);
        on("lse", t, geo.device);
        lse = t.data_ptr<float>();
    }
    const double scale = PyFloat_AsDouble(a[8]);
    const int causal = PyObject_IsTrue(a[9]);
    if (causal < 0 || PyErr_Occurred()) throw Refused();
    check(ffnrm_kv_attend(geo.kv, int32_of("layer", integer(a[1])), &batch, dtype, &qr, &yr, lse, int32_of("heads", heads), float(scale),
                          causal, int32_of("window", integer(a[10])), stream.ptr));
    stream.keep({a[2], a[3], a[4], a[5], a[6], a[7]});
    written(a[6]);
    written(a[7]);
    return THPVariable_Wrap(std::move(out));
}

// geo, layer, tables, lengths, starts, rows, element type, stream
PyObject *read(PyObject *const *a) {
    const Geo geo(a[0]);
    const Stream stream(a[7], geo.device);
    const int64_t rows = integer(a[5]), dtype = integer(a[6]);
    const at::ScalarType type = dtype == FFNRM_F16 ? at::kHalf : dtype == FFNRM_BF16 ? at::kBFloat16 : at::kFloat;
    if (rows < 0) refuse("rows=%lld must not be negative", (long long)rows);
    const ffnrm_kv_batch batch = batch_of(a[2], a[3], a[4], rows, geo.device);
    at::Tensor k = empty({rows, geo.heads, geo.dim}, type, geo.device), v = empty({rows, geo.heads, geo.dim}, type, geo.device);
    check(ffnrm_kv_read(geo.kv, int32_of("layer", integer(a[1])), &batch, int(dtype), k.data_ptr(), v.data_ptr(), stream.ptr));
    stream.keep({a[2], a[3], a[4]});
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
}

at::Tensor given_or(PyObject *o, const char *name, at::IntArrayRef shape, int device) {
    return o == Py_None ? empty(shape, at::kInt, device) : tensor(name, o);
}

// geo, tables, lengths, parents, extra, out_tables or None, out_lengths or None, info or None, stream
PyObject *fork(PyObject *const *a) {
    const Geo geo(a[0]);
    const int d = geo.device;
    const Stream stream(a[8], d);
    const at::Tensor &t = tensor("tables", a[1]), &parents = tensor("parents", a[3]);
    if (t.dim() != 2 || parents.dim() != 1) refuse("tables must have shape (seqs, width), parents (children,)");
    const int64_t n = parents.size(0);
    at::Tensor out = given_or(a[5], "out_tables", {n, t.size(1)}, d), lens = given_or(a[6], "out_lengths", {n}, d),
               info = given_or(a[7], "info", {4}, d);
    if (out.dim() != 2 || out.size(0) != n) refuse("out_tables must have shape (children, width)");
    check(ffnrm_kv_fork(geo.kv, ints("tables", t, d), ints1("lengths", tensor("lengths", a[2]), t.size(0), d), int32_of("seqs", t.size(0)),
                        int32_of("width", t.size(1)), ints1("parents", parents, n, d), ints1("extra", tensor("extra", a[4]), n, d),
                        int32_of("children", n), ints("out_tables", out, d), int32_of("width", out.size(1)),
                        ints1("out_lengths", lens, n, d), ints1("info", info, 4, d), stream.ptr));
    stream.keep({a[1], a[2], a[3], a[4], a[5], a[6], a[7]});
    for (int i : {5, 6, 7}) written(a[i]);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lens)), THPVariable_Wrap(std::move(info)));
}

// geo, tables, lengths, out_tables or None, info or None, stream
PyObject *compact(PyObject *const *a) {
    const Geo geo(a[0]);
    const int d = geo.device;
    const Stream stream(a[5], d);
    const at::Tensor &t = tensor("tables", a[1]);
    if (t.dim() != 2) refuse("tables must have shape (seqs, width)");
    at::Tensor out = given_or(a[3], "out_tables", {t.size(0), t.size(1)}, d), info = given_or(a[4], "info", {4}, d);
    if (out.sizes() != t.sizes()) refuse("out_tables must have tables' shape");
    check(ffnrm_kv_compact(geo.kv, ints("tables", t, d), ints1("lengths", tensor("lengths", a[2]), t.size(0), d),
                           int32_of("seqs", t.size(0)), int32_of("width", t.size(1)), ints("out_tables", out, d),
                           ints1("info", info, 4, d), stream.ptr));
    stream.keep({a[1], a[2], a[3], a[4]});
    for (int i : {3, 4}) written(a[i]);
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(info)));
}

// geo, src, dst, stream
PyObject *copy_pages(PyObject *const *a) {
    const Geo geo(a[0]);
    const Stream stream(a[3], geo.device);
    const at::Tensor &src = tensor("src", a[1]);
    if (src.dim() != 1) refuse("src must have shape (n,)");
    check(ffnrm_kv_copy_pages(geo.kv, ints("src", src, geo.device), ints1("dst", tensor("dst", a[2]), src.size(0), geo.device),
                              int32_of("n", src.size(0)), stream.ptr));
    stream.keep({a[1], a[2]});
    Py_RETURN_NONE;
}

#define BIND(NAME, N) \
    PyObject *py_##NAME(PyObject *, PyObject *const *args, Py_ssize_t n) { return guarded<NAME>(args, n, N); }
BIND(rotary, 6)
BIND(append, 12)
BIND(attend, 12)
BIND(read, 8)
BIND(fork, 9)
BIND(compact, 6)
BIND(copy_pages, 4)
#define ENTRY(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(rotary), ENTRY(append), ENTRY(attend), ENTRY(read), ENTRY(fork), ENTRY(compact), ENTRY(copy_pages),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ffnrm_kv_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_ffnrm_kv_bind() { return PyModule_Create(&module); }
