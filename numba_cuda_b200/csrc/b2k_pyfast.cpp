// Python extension `_pyfast`: the head-wise calls (kernels/headnorm.py, kernels/kvcache.py)
// for the common arguments, torch tensors with outputs given, without the
// interpreter's time for ten tensors' attributes (a call's host time 14 -> 6.5 us).
//
// Every function here reads its arguments and either makes the C-ABI call and returns its
// status, or returns None without having done anything -- for any argument that is not
// a plain tensor and for anything that looks wrong.  The Python code then runs from the
// start and is the only place where arguments are converted and errors are raised.
// What is accepted here is therefore a subset of what it accepts.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <initializer_list>

#include "../../include/b2k.h"

namespace {

// Set once by setup().
PyObject *g_tensor_type, *g_formats, *g_stream_ptr, *g_workspace, *g_forward_mode, *g_level, *g_written, *g_no_arguments;

// An attribute or a method without arguments of the tensor type.  Where it is implemented
// in C, its function is called directly: looking six of them up for each of ten tensors
// was a fifth of a call's host time.
struct Member {
    const char *name;
    PyObject *key = nullptr;
    bool called = false;                  // a method
    getter get = nullptr;
    void *closure = nullptr;
    PyCFunction plain = nullptr;          // METH_NOARGS
    PyCFunctionWithKeywords keyed = nullptr;

    bool find(PyObject *type) {
        Py_XSETREF(key, PyUnicode_InternFromString(name));
        PyObject *d = key ? PyObject_GetAttr(type, key) : nullptr;       // held for good: the pointers live in it
        if (d == nullptr) return false;
        get = nullptr;
        plain = nullptr;
        keyed = nullptr;
        called = !Py_IS_TYPE(d, &PyGetSetDescr_Type) && PyCallable_Check(d);
        if (Py_IS_TYPE(d, &PyGetSetDescr_Type)) {
            const PyGetSetDef *def = reinterpret_cast<PyGetSetDescrObject *>(d)->d_getset;
            get = def->get;
            closure = def->closure;
        } else if (Py_IS_TYPE(d, &PyMethodDescr_Type)) {
            const PyMethodDef *def = reinterpret_cast<PyMethodDescrObject *>(d)->d_method;
            if (def->ml_flags == METH_NOARGS) plain = def->ml_meth;
            else if (def->ml_flags == (METH_VARARGS | METH_KEYWORDS))
                keyed = reinterpret_cast<PyCFunctionWithKeywords>(reinterpret_cast<void (*)()>(def->ml_meth));
        }
        return true;
    }
    PyObject *operator()(PyObject *o) const {
        if (get) return get(o, closure);
        if (plain) return plain(o, nullptr);
        if (keyed) return keyed(o, g_no_arguments, nullptr);
        if (!called) return PyObject_GetAttr(o, key);
        PyObject *args[1] = {o};
        return PyObject_VectorcallMethod(key, args, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, nullptr);
    }
};
Member m_dtype{"dtype"}, m_shape{"shape"}, m_stride{"stride"}, m_data_ptr{"data_ptr"}, m_get_device{"get_device"},
    m_requires_grad{"requires_grad"};

struct Entry {
    decltype(&b2k_norm_rotate) norm_rotate;
    decltype(&b2k_norm_rotate_backward_scratch_bytes) scratch_bytes;
    decltype(&b2k_norm_rotate_backward) norm_rotate_backward;
    decltype(&b2k_cache_write) cache_write;
    decltype(&b2k_cache_read) cache_read;
    decltype(&b2k_norm_rotate_write) norm_rotate_write;
    decltype(&b2k_current_device) current_device;
} g_call;

struct Array {
    void *data;
    long long size[4], stride[4];
    int ndim, format, device;
};

bool as_integer(PyObject *o, long long &v) {            // takes the reference
    if (o == nullptr) return false;
    v = PyLong_AsLongLong(o);
    Py_DECREF(o);
    return !(v == -1 && PyErr_Occurred());
}

bool integers(PyObject *tuple, long long *out, int &n) {  // takes the reference
    if (tuple == nullptr) return false;
    bool ok = PyTuple_Check(tuple) && PyTuple_GET_SIZE(tuple) <= 4;
    if (ok) {
        n = static_cast<int>(PyTuple_GET_SIZE(tuple));
        for (int i = 0; i < n && ok; ++i) {
            out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
            ok = !(out[i] == -1 && PyErr_Occurred());
        }
    }
    Py_DECREF(tuple);
    return ok;
}

// A plain tensor on the current device that does not require grad.  False may leave a
// Python error behind; the entry points clear it.
bool read(PyObject *o, int device, Array &a) {
    if (reinterpret_cast<PyObject *>(Py_TYPE(o)) != g_tensor_type) return false;
    PyObject *dtype = m_dtype(o);
    if (dtype == nullptr) return false;
    PyObject *format = PyDict_GetItemWithError(g_formats, dtype);      // borrowed
    Py_DECREF(dtype);
    if (format == nullptr) return false;
    a.format = static_cast<int>(PyLong_AsLong(format));
    PyObject *grad = m_requires_grad(o);
    if (grad == nullptr) return false;
    const bool plain = grad == Py_False;
    Py_DECREF(grad);
    if (!plain) return false;
    long long v;
    if (!as_integer(m_get_device(o), v) || v != device) return false;
    a.device = device;
    if (!as_integer(m_data_ptr(o), v)) return false;
    a.data = reinterpret_cast<void *>(v);
    int strides = 0;
    if (!integers(m_shape(o), a.size, a.ndim)) return false;
    return integers(m_stride(o), a.stride, strides) && strides == a.ndim;
}

bool is_float(int format) { return format == B2K_FMT_F32 || format == B2K_FMT_F16 || format == B2K_FMT_BF16; }
bool is_index(int format) { return format == B2K_FMT_I32 || format == B2K_FMT_I64; }
int index_bytes(const Array &a) { return a.format == B2K_FMT_I32 ? 4 : 8; }

// (tokens, heads, dim) of floats
bool read_heads(PyObject *o, int device, Array &a, b2k_heads &h) {
    if (!read(o, device, a) || a.ndim != 3 || !is_float(a.format) || (a.stride[2] != 1 && a.size[2] > 1)) return false;
    h = b2k_heads{a.data, a.stride[0], a.stride[1], a.size[1], a.size[2]};
    return true;
}

bool read_vector(PyObject *o, int device, long long length, Array &a) {
    return read(o, device, a) && a.ndim == 1 && a.size[0] == length && (a.stride[0] == 1 || length <= 1);
}

bool same_shape(const Array &a, const Array &b) {
    if (a.ndim != b.ndim || a.format != b.format) return false;
    for (int i = 0; i < a.ndim; ++i)
        if (a.size[i] != b.size[i]) return false;
    return true;
}

// An output of an input's shape and type; `given` says whether the input is there.
bool read_result(PyObject *o, bool given, const Array &like, int device, b2k_heads &h) {
    h = b2k_heads{};
    if (!given) return o == Py_None;
    Array a;
    return read_heads(o, device, a, h) && same_shape(a, like);
}

struct Rotation {
    b2k_rotation r{};
    Array q, k;
    bool has_q = false, has_k = false;
    const Array &first() const { return has_q ? q : k; }
};

bool truth(PyObject *o, int64_t &v) {
    if (o != Py_True && o != Py_False) return false;
    v = o == Py_True;
    return true;
}

// q, k, q_weight, k_weight, cos, sin, positions of args[0..7)
bool read_rotation(PyObject *const *args, PyObject *eps, PyObject *interleaved, PyObject *norm, int device, Rotation &t) {
    t.has_q = args[0] != Py_None;
    t.has_k = args[1] != Py_None;
    if (!t.has_q && !t.has_k) return false;
    if (t.has_q && !read_heads(args[0], device, t.q, t.r.q)) return false;
    if (t.has_k && !read_heads(args[1], device, t.k, t.r.k)) return false;
    if (t.has_q && t.has_k && (t.q.size[0] != t.k.size[0] || t.q.format != t.k.format)) return false;
    if (!truth(interleaved, t.r.interleaved) || !truth(norm, t.r.norm)) return false;
    t.r.eps = PyFloat_AsDouble(eps);
    if (t.r.eps == -1.0 && PyErr_Occurred()) return false;
    t.r.format = t.first().format;
    t.r.tokens = t.first().size[0];
    t.r.weight_format = B2K_FMT_F32;
    const void **weight[2] = {&t.r.q_weight_dev, &t.r.k_weight_dev};
    int weights = 0;
    for (int i = 0; i < 2; ++i) {
        PyObject *o = args[2 + i];
        if (o == Py_None) continue;
        Array a;
        if (!(i ? t.has_k : t.has_q) || !t.r.norm) return false;
        if (!read_vector(o, device, i ? t.k.size[2] : t.q.size[2], a) || !is_float(a.format)) return false;
        if (weights++ && a.format != t.r.weight_format) return false;
        t.r.weight_format = a.format;
        *weight[i] = a.data;
    }
    t.r.position_bytes = 8;
    if (args[4] == Py_None && args[5] == Py_None && args[6] == Py_None) return true;
    Array c, s, at;
    if (!read(args[4], device, c) || !read(args[5], device, s) || !read_vector(args[6], device, t.r.tokens, at)) return false;
    if (c.format != B2K_FMT_F32 || c.ndim != 2 || !same_shape(c, s) || !is_index(at.format)) return false;
    if (c.size[1] > 1 && (c.stride[1] != 1 || s.stride[1] != 1)) return false;
    if ((t.has_q && 2 * c.size[1] > t.q.size[2]) || (t.has_k && 2 * c.size[1] > t.k.size[2])) return false;
    t.r.rotary_dim = 2 * c.size[1];
    t.r.cos_dev = static_cast<const float *>(c.data);
    t.r.sin_dev = static_cast<const float *>(s.data);
    t.r.cos_stride = c.stride[0];
    t.r.sin_stride = s.stride[0];
    t.r.table_rows = c.size[0];
    t.r.positions_dev = at.data;
    t.r.position_bytes = index_bytes(at);
    return true;
}

// k_codes, k_scales, v_codes, v_scales of args[0..4); the codes' types or `format` tell what they
// are.  `given` says which sides are there.
bool read_cache(PyObject *const *args, PyObject *format, int device, b2k_cache &c, bool (&given)[2]) {
    int code = -1;
    if (format != Py_None) {
        if (!PyUnicode_CheckExact(format)) return false;
        if (PyUnicode_CompareWithASCIIString(format, "e4m3") == 0) code = B2K_FMT_E4M3;
        else if (PyUnicode_CompareWithASCIIString(format, "e5m2") == 0) code = B2K_FMT_E5M2;
        else return false;
    }
    c = b2k_cache{};
    b2k_pages *side[2] = {&c.k, &c.v};
    bool any = false;
    for (int i = 0; i < 2; ++i) {
        PyObject *codes = args[2 * i], *scales = args[2 * i + 1];
        given[i] = codes != Py_None || scales != Py_None;
        if (!given[i]) continue;
        Array a, s;
        if (!read(codes, device, a) || !read(scales, device, s) || a.ndim != 4 || s.ndim != 4) return false;
        if (a.format == B2K_FMT_E4M3 || a.format == B2K_FMT_E5M2) {
            if (code >= 0 && code != a.format) return false;
            code = a.format;
        } else if (a.format != B2K_FMT_U8) {
            return false;
        }
        if (s.format == B2K_FMT_U8) s.format = B2K_FMT_E8M0;
        if (s.format != B2K_FMT_F32 && s.format != B2K_FMT_E8M0) return false;
        for (int j = 0; j < 3; ++j)
            if (a.size[j] != s.size[j]) return false;
        if ((a.stride[3] != 1 && a.size[3] > 1) || (s.stride[3] != 1 && s.size[3] > 1)) return false;
        if (s.size[3] < 1 || a.size[3] % s.size[3]) return false;
        if (any && (c.scale_format != s.format || c.pages != a.size[0] || c.page_size != a.size[1])) return false;
        any = true;
        c.scale_format = s.format;
        c.pages = a.size[0];
        c.page_size = a.size[1];
        *side[i] = b2k_pages{a.data, a.stride[0], a.stride[1], a.stride[2], s.data, s.stride[0], s.stride[1], s.stride[2],
                             a.size[2], a.size[3], a.size[3] / s.size[3]};
    }
    c.code_format = code < 0 ? B2K_FMT_E4M3 : code;
    return any;
}

// An array and its side of the cache: both are there and alike, or neither is.
bool fits(bool given, const b2k_heads &h, bool side_given, const b2k_pages &side) {
    return given == side_given && (!given || (h.heads == side.heads && h.dim == side.dim && side.dim > 0));
}

bool read_stream(PyObject *o, void *&stream) {
    long long v;
    if (PyLong_CheckExact(o)) {
        v = PyLong_AsLongLong(o);
        if (v == -1 && PyErr_Occurred()) return false;
    } else if (!as_integer(PyObject_CallOneArg(g_stream_ptr, o), v)) {
        return false;
    }
    stream = reinterpret_cast<void *>(v);
    return true;
}

PyObject *pass() {                  // let the Python code look at it
    PyErr_Clear();
    Py_RETURN_NONE;
}

bool ready(Py_ssize_t given, Py_ssize_t wanted, int &device) {
    if (g_tensor_type == nullptr || given != wanted) return false;
    // inside a level of forward differentiation a tensor may carry a tangent: the Python code looks
    PyObject *level = PyDict_GetItemWithError(g_forward_mode, g_level);             // borrowed
    if (level == nullptr || PyLong_AsLong(level) != -1 || PyErr_Occurred()) return false;
    device = g_call.current_device();
    return device >= 0;
}

// Makes the call `f` without the interpreter lock: a launch waits when the GPU's queue is full.  The
// arguments are held by the caller of the entry point meanwhile.
template <typename F>
int unlocked(F f) {
    PyThreadState *state = PyEval_SaveThread();
    const int status = f();
    PyEval_RestoreThread(state);
    return status;
}

// The status of a call; after a good one autograd is told which tensors (or None) it has written.
PyObject *done(int status, std::initializer_list<PyObject *> outputs) {
    if (status == 0) {
        Py_ssize_t n = 0;
        for (PyObject *o : outputs) n += o != Py_None;
        PyObject *tensors = PyTuple_New(n);
        if (tensors == nullptr) return nullptr;
        n = 0;
        for (PyObject *o : outputs)
            if (o != Py_None) PyTuple_SET_ITEM(tensors, n++, Py_NewRef(o));
        PyObject *none = PyObject_CallOneArg(g_written, tensors);
        Py_DECREF(tensors);
        if (none == nullptr) return nullptr;
        Py_DECREF(none);
    }
    return PyLong_FromLong(status);
}

// (q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, q_out, k_out, stream)
PyObject *norm_rotate(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int device;
    Rotation t;
    b2k_heads q_out, k_out;
    void *stream;
    if (!ready(n, 13, device) || !read_rotation(args, args[7], args[8], args[9], device, t) ||
        !read_result(args[10], t.has_q, t.q, device, q_out) || !read_result(args[11], t.has_k, t.k, device, k_out) ||
        !read_stream(args[12], stream))
        return pass();
    return done(unlocked([&] { return g_call.norm_rotate(&t.r, &q_out, &k_out, stream); }), {args[10], args[11]});
}

// (q, k, q_weight, k_weight, cos, sin, positions, q_grad, k_grad, eps, interleaved, norm, dq, dk, dq_weight, dk_weight, stream)
PyObject *norm_rotate_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int device;
    Rotation t;
    b2k_heads q_grad, k_grad, dq, dk;
    void *stream;
    if (!ready(n, 17, device) || !read_rotation(args, args[9], args[10], args[11], device, t) ||
        !read_result(args[7], t.has_q, t.q, device, q_grad) || !read_result(args[8], t.has_k, t.k, device, k_grad) ||
        !read_result(args[12], t.has_q, t.q, device, dq) || !read_result(args[13], t.has_k, t.k, device, dk) ||
        !read_stream(args[16], stream))
        return pass();
    void *sums[2] = {};
    for (int i = 0; i < 2; ++i) {
        const bool given = (i ? t.r.k_weight_dev : t.r.q_weight_dev) != nullptr;
        if (given != (args[2 + i] != Py_None)) return pass();          // a weight without memory
        if (!given) {
            if (args[14 + i] != Py_None) return pass();
            continue;
        }
        Array a;
        if (!read_vector(args[14 + i], device, i ? t.k.size[2] : t.q.size[2], a) || a.format != t.r.weight_format) return pass();
        sums[i] = a.data;
    }
    PyObject *held = nullptr;
    void *scratch = nullptr;
    long long bytes = 0;
    if (sums[0] || sums[1]) {
        bytes = g_call.scratch_bytes(&t.r);
        PyObject *size = PyLong_FromLongLong(bytes);
        if (size == nullptr) return pass();
        PyObject *const two[2] = {size, args[16]};
        held = PyObject_Vectorcall(g_workspace, two, 2, nullptr);
        Py_DECREF(size);
        if (held == nullptr) return nullptr;                            // out of memory, say
        Array scratch_of;
        if (!read(held, device, scratch_of)) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "no workspace tensor");
            Py_DECREF(held);
            return nullptr;
        }
        scratch = scratch_of.data;
    }
    const int status = unlocked([&] {
        return g_call.norm_rotate_backward(&t.r, &q_grad, &k_grad, &dq, &dk, sums[0], sums[1], scratch, bytes, stream);
    });
    Py_XDECREF(held);
    return done(status, {args[12], args[13], args[14], args[15]});
}

// (k, v, k_codes, k_scales, v_codes, v_scales, slots, format, stream)
PyObject *cache_write(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int device;
    b2k_cache cache;
    bool side[2];
    b2k_heads h[2] = {};
    Array a[2], at;
    void *stream;
    if (!ready(n, 9, device) || !read_cache(args + 2, args[7], device, cache, side)) return pass();
    const bool has[2] = {args[0] != Py_None, args[1] != Py_None};
    for (int i = 0; i < 2; ++i)
        if ((has[i] && !read_heads(args[i], device, a[i], h[i])) || !fits(has[i], h[i], side[i], i ? cache.v : cache.k)) return pass();
    if (has[0] && has[1] && (a[0].size[0] != a[1].size[0] || a[0].format != a[1].format)) return pass();
    const Array &first = has[0] ? a[0] : a[1];
    if (!(has[0] || has[1]) || !read_vector(args[6], device, first.size[0], at) || !is_index(at.format) ||
        !read_stream(args[8], stream))
        return pass();
    const int status = unlocked([&] {
        return g_call.cache_write(&cache, first.format, first.size[0], &h[0], &h[1], at.data, index_bytes(at), stream);
    });
    return done(status, {args[2], args[3], args[4], args[5]});
}

// (k_codes, k_scales, v_codes, v_scales, page_table, offsets, k_out, v_out, format, stream)
PyObject *cache_read(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int device;
    b2k_cache cache;
    bool side[2];
    b2k_heads h[2] = {};
    Array a[2], table, at;
    void *stream;
    if (!ready(n, 10, device) || !read_cache(args, args[8], device, cache, side)) return pass();
    const bool has[2] = {args[6] != Py_None, args[7] != Py_None};
    for (int i = 0; i < 2; ++i)
        if ((has[i] && !read_heads(args[6 + i], device, a[i], h[i])) || !fits(has[i], h[i], side[i], i ? cache.v : cache.k)) return pass();
    if (has[0] && has[1] && (a[0].size[0] != a[1].size[0] || a[0].format != a[1].format)) return pass();
    const Array &first = has[0] ? a[0] : a[1];
    if (!(has[0] || has[1]) || !read(args[4], device, table) || table.ndim != 2 || !is_index(table.format) ||
        (table.stride[1] != 1 && table.size[1] > 1) || !read_vector(args[5], device, table.size[0] + 1, at) ||
        !is_index(at.format) || !read_stream(args[9], stream))
        return pass();
    const int status = unlocked([&] {
        return g_call.cache_read(&cache, first.format, first.size[0], &h[0], &h[1], table.data, table.stride[0], table.size[1],
                                 index_bytes(table), at.data, table.size[0], index_bytes(at), stream);
    });
    return done(status, {args[6], args[7]});
}

// (q, k, q_weight, k_weight, cos, sin, positions, v, k_codes, k_scales, v_codes, v_scales, slots, eps, interleaved, norm,
//  format, q_out, stream)
PyObject *norm_rotate_write(PyObject *, PyObject *const *args, Py_ssize_t n) {
    int device;
    Rotation t;
    b2k_cache cache;
    bool side[2];
    b2k_heads v{}, q_out;
    Array av, at;
    void *stream;
    if (!ready(n, 19, device) || !read_rotation(args, args[13], args[14], args[15], device, t) ||
        !read_cache(args + 8, args[16], device, cache, side) || !read_result(args[17], t.has_q, t.q, device, q_out))
        return pass();
    const bool has_v = args[7] != Py_None;
    if (has_v && (!read_heads(args[7], device, av, v) || av.size[0] != t.r.tokens || av.format != t.r.format)) return pass();
    if (!fits(t.has_k, t.r.k, side[0], cache.k) || !fits(has_v, v, side[1], cache.v) || !read_vector(args[12], device, t.r.tokens, at) ||
        !is_index(at.format) || !read_stream(args[18], stream))
        return pass();
    const int status =
        unlocked([&] { return g_call.norm_rotate_write(&t.r, &v, &q_out, &cache, at.data, index_bytes(at), stream); });
    return done(status, {args[17], args[8], args[9], args[10], args[11]});
}

template <typename F>
bool address(PyObject *dict, const char *name, F &f) {
    PyObject *o = PyDict_GetItemString(dict, name);                 // borrowed
    if (o == nullptr) {
        PyErr_Format(PyExc_KeyError, "no address of %s", name);
        return false;
    }
    f = reinterpret_cast<F>(PyLong_AsVoidPtr(o));
    return !PyErr_Occurred();
}

// setup(tensor type, {dtype: format}, {entry point: address}, stream_ptr, workspace, names of torch.autograd.forward_ad,
//       function to call with a tuple of written tensors)
PyObject *setup(PyObject *, PyObject *args) {
    PyObject *type, *formats, *addresses, *stream, *workspace, *forward, *written;
    if (!PyArg_ParseTuple(args, "OO!O!OOO!O", &type, &PyDict_Type, &formats, &PyDict_Type, &addresses, &stream, &workspace,
                          &PyDict_Type, &forward, &written))
        return nullptr;
    Entry e;
    if (!address(addresses, "b2k_norm_rotate", e.norm_rotate) ||
        !address(addresses, "b2k_norm_rotate_backward_scratch_bytes", e.scratch_bytes) ||
        !address(addresses, "b2k_norm_rotate_backward", e.norm_rotate_backward) ||
        !address(addresses, "b2k_cache_write", e.cache_write) || !address(addresses, "b2k_cache_read", e.cache_read) ||
        !address(addresses, "b2k_norm_rotate_write", e.norm_rotate_write) ||
        !address(addresses, "b2k_current_device", e.current_device))
        return nullptr;
    for (Member *m : {&m_dtype, &m_shape, &m_stride, &m_data_ptr, &m_get_device, &m_requires_grad})
        if (!m->find(type)) return nullptr;
    g_call = e;
    Py_INCREF(formats);
    Py_XSETREF(g_formats, formats);
    Py_INCREF(stream);
    Py_XSETREF(g_stream_ptr, stream);
    Py_INCREF(workspace);
    Py_XSETREF(g_workspace, workspace);
    Py_INCREF(written);
    Py_XSETREF(g_written, written);
    Py_INCREF(forward);
    Py_XSETREF(g_forward_mode, forward);
    Py_INCREF(type);
    Py_XSETREF(g_tensor_type, type);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef g_methods[] = {
    {"setup", setup, METH_VARARGS, "Give the module the tensor type, the formats and the library's entry points."},
    {"norm_rotate", FAST(norm_rotate), METH_FASTCALL, nullptr},
    {"norm_rotate_backward", FAST(norm_rotate_backward), METH_FASTCALL, nullptr},
    {"cache_write", FAST(cache_write), METH_FASTCALL, nullptr},
    {"cache_read", FAST(cache_read), METH_FASTCALL, nullptr},
    {"norm_rotate_write", FAST(norm_rotate_write), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_pyfast", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pyfast(void) {
    g_no_arguments = PyTuple_New(0);
    g_level = PyUnicode_InternFromString("_current_level");
    if (g_no_arguments == nullptr || g_level == nullptr) return nullptr;
    return PyModule_Create(&g_module);
}
