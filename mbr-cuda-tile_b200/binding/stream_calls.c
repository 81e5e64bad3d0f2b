/* stream_calls.c — the streaming operators' calls from Python.
 *
 * A frame's kernels take two or three microseconds; checking six to ten tensors
 * and converting twenty arguments in Python takes several times that.  This
 * extension does the same work through the C API: it looks at each tensor once
 * (stride, shape, dtype, device, address, by torch's public attributes), checks it,
 * allocates the outputs with torch and calls the library's entry points, whose
 * addresses cudasep.py hands over once (bind).  It holds no state beyond what
 * bind was given. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/mbr_b200.h"

/* ---- what bind() is given ---- */
static int (*f_norm)(const mbr_view*, const mbr_view*, const mbr_view*, const mbr_view*, int64_t, int64_t, int, int, int,
                     const float*, const float*, float, const float*, const float*, int64_t, const int32_t*, int,
                     const int*, int, void*);
static int (*f_append)(const mbr_kv_cache*, const mbr_view*, const mbr_view*, const int32_t*, const int32_t*, int64_t,
                       void*);
static int (*f_read)(const mbr_kv_cache*, const int32_t*, const int32_t*, int64_t, const mbr_view*, const mbr_view*,
                     void*);
static int (*f_window)(const mbr_view*, const mbr_view*, const mbr_view*, const mbr_view*, int64_t, int64_t, int64_t, int,
                       int, int, const int32_t*, const int32_t*, int, int, int, float, const float*, int, void*, int64_t,
                       void*);
static int (*f_window_ws)(int64_t, int64_t, int64_t, int, int, int, int, int, int, int, int64_t*);
static int (*f_cache)(const mbr_view*, const mbr_kv_cache*, const mbr_view*, const int32_t*, int64_t, int, int, int, float,
                      const float*, void*, int64_t, void*);
static int (*f_cache_ws)(const mbr_kv_cache*, int64_t, int, int, int, int64_t*);
static PyObject *t_f32, *t_i32, *t_u8;    /* torch dtypes */
static PyObject* t_codes;                 /* {dtype: code} */
static PyObject *p_empty_like, *p_kwargs; /* torch.empty_like and {"memory_format": torch.contiguous_format} */
static PyObject *p_stream, *p_device;     /* current stream's handle of a device; current device */
static PyObject *p_check, *p_elsewhere, *p_workspace, *p_like_on;
static PyObject *s_stride, *s_shape, *s_dtype, *s_get_device, *s_data_ptr, *s_contiguous, *s_device, *s_desc, *s_dev,
    *s_new, *s_cuda_stream, *s_cache_dtype;

/* ---- looking at tensors ---- */
typedef struct {
    mbr_view v;
    int64_t n[4];
} rows_t;

static int is_dtype(PyObject* t, PyObject* dtype) {
    PyObject* d = PyObject_GetAttr(t, s_dtype);
    if (!d) return -1;
    Py_DECREF(d); /* dtypes are singletons that torch keeps */
    return d == dtype;
}

static int long_method(PyObject* t, PyObject* name, long long* out) {
    PyObject* r = PyObject_CallMethodNoArgs(t, name);
    if (!r) return -1;
    *out = PyLong_AsLongLong(r);
    Py_DECREF(r);
    return *out == -1 && PyErr_Occurred() ? -1 : 0;
}

static int address(PyObject* t, void** out) {
    PyObject* r = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (!r) return -1;
    *out = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return !*out && PyErr_Occurred() ? -1 : 0;
}

/* Sizes of a tensor's shape (up to most); the number of axes, or -1. */
static Py_ssize_t sizes(PyObject* t, PyObject* name, int call, int64_t* n, Py_ssize_t most) {
    PyObject* s = call ? PyObject_CallMethodNoArgs(t, name) : PyObject_GetAttr(t, name);
    Py_ssize_t k = -1;
    if (s && PyTuple_Check(s)) {
        k = PyTuple_GET_SIZE(s);
        for (Py_ssize_t i = 0; i < k && i < most; ++i) n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(s, i));
    } else if (s) {
        PyErr_SetString(PyExc_ValueError, "expected a tensor");
    }
    Py_XDECREF(s);
    return PyErr_Occurred() ? -1 : k;
}

static int bad_rows(const char* name, PyObject* t, PyObject* dtype, long long dev) {
    if (!PyErr_Occurred()) {
        PyObject *sh = PyObject_GetAttr(t, s_shape), *dt = PyObject_GetAttr(t, s_dtype), *dv = PyObject_GetAttr(t, s_device);
        if (sh && dt && dv)
            PyErr_Format(PyExc_ValueError,
                         "%s must be [seqs, tokens, heads, dim_head] of %S on cuda:%lld with a contiguous last axis, "
                         "got %S of %S on %S",
                         name, dtype, dev, sh, dt, dv);
        Py_XDECREF(sh), Py_XDECREF(dt), Py_XDECREF(dv);
    }
    return -1;
}

static int rows(const char* name, PyObject* t, PyObject* dtype, long long dev, rows_t* r) {
    int64_t st[4];
    long long d;
    int same;
    if (sizes(t, s_stride, 1, st, 4) != 4 || sizes(t, s_shape, 0, r->n, 4) != 4 || (same = is_dtype(t, dtype)) < 0 ||
        !same || long_method(t, s_get_device, &d) || d != dev || (st[3] != 1 && r->n[3] > 1))
        return bad_rows(name, t, dtype, dev);
    r->v.seq = st[0], r->v.token = st[1], r->v.head = st[2];
    return address(t, &r->v.data);
}

/* A contiguous tensor of this type and shape, or None. */
static int flat(const char* name, PyObject* t, PyObject* dtype, long long dev, Py_ssize_t k, const int64_t* n, void** out) {
    *out = NULL;
    if (t == Py_None) return 0;
    int64_t got[5];
    long long d = -1;
    int ok = sizes(t, s_shape, 0, got, 5) == k && is_dtype(t, dtype) == 1 && !long_method(t, s_get_device, &d) && d == dev;
    for (Py_ssize_t i = 0; ok && i < k; ++i) ok = got[i] == n[i];
    if (ok) {
        PyObject* c = PyObject_CallMethodNoArgs(t, s_contiguous);
        ok = c == Py_True;
        Py_XDECREF(c);
    }
    if (ok) return address(t, out);
    if (!PyErr_Occurred()) {
        PyObject *sh = PyObject_GetAttr(t, s_shape), *dt = PyObject_GetAttr(t, s_dtype), *dv = PyObject_GetAttr(t, s_device);
        PyObject* want = PyTuple_New(k);
        for (Py_ssize_t i = 0; want && i < k; ++i) PyTuple_SET_ITEM(want, i, PyLong_FromLongLong(n[i]));
        if (sh && dt && dv && want)
            PyErr_Format(PyExc_ValueError, "%s must be contiguous %S of shape %S on cuda:%lld, got %S of %S on %S", name,
                         dtype, want, dev, sh, dt, dv);
        Py_XDECREF(sh), Py_XDECREF(dt), Py_XDECREF(dv), Py_XDECREF(want);
    }
    return -1;
}

static int refuse(const char* text) {
    PyErr_SetString(PyExc_ValueError, text);
    return -1;
}

static int code_of(PyObject* dtype) {
    PyObject* c = PyDict_GetItemWithError(t_codes, dtype);
    if (!c) {
        if (!PyErr_Occurred())
            PyErr_Format(PyExc_ValueError, "dtype must be float32, float16 or bfloat16, got %S", dtype);
        return -1;
    }
    return (int)PyLong_AsLong(c);
}

static int device_of(PyObject* t, long long* dev) {
    if (long_method(t, s_get_device, dev)) return -1;
    return *dev >= 0 ? 0 : refuse("tensors must be on a CUDA device");
}

/* New contiguous tensor of the same shape and type, the memory of `stream` (None: the current one). */
static PyObject* like(PyObject* t, PyObject* stream) {
    PyObject* args[2] = {t, stream};
    return stream == Py_None ? PyObject_VectorcallDict(p_empty_like, args, 1, p_kwargs)
                             : PyObject_Vectorcall(p_like_on, args, 2, NULL);
}

/* 1: `dev` is current and *handle is the stream to use; 0: another device is current; -1: error. */
static int stream_of(PyObject* stream, long long dev, void** handle) {
    PyObject* cur = PyObject_CallNoArgs(p_device);
    if (!cur) return -1;
    const long long now = PyLong_AsLongLong(cur);
    Py_DECREF(cur);
    if (now != dev) return PyErr_Occurred() ? -1 : 0;
    PyObject* h;
    if (stream == Py_None) {
        PyObject* d = PyLong_FromLongLong(dev);
        h = d ? PyObject_CallOneArg(p_stream, d) : NULL;
        Py_XDECREF(d);
    } else if (PyLong_Check(stream)) {
        h = Py_NewRef(stream);
    } else {
        h = PyObject_GetAttr(stream, s_cuda_stream);
    }
    if (!h) return -1;
    *handle = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    return PyErr_Occurred() ? -1 : 1;
}

/* The call once more with `dev` current (cudasep.py enters it). */
static PyObject* elsewhere(long long dev, const char* name, PyObject* const* args, Py_ssize_t n) {
    PyObject* a = PyTuple_New(n);
    if (!a) return NULL;
    for (Py_ssize_t i = 0; i < n; ++i) PyTuple_SET_ITEM(a, i, Py_NewRef(args[i]));
    PyObject* r = PyObject_CallFunction(p_elsewhere, "LsO", dev, name, a);
    Py_DECREF(a);
    return r;
}

static int checked(int rc) { /* cudasep's exception for a status code */
    if (rc == 0) return 0;
    PyObject* r = PyObject_CallFunction(p_check, "i", rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the library refused the call");
    return -1;
}

static int int_arg(PyObject* o, int* out) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (!PyErr_ExceptionMatches(PyExc_OverflowError)) return -1;
        PyErr_Clear();
        *out = 1 << 30;
        return 0;
    }
    *out = v >= (1 << 30) ? 1 << 30 : v < -(1 << 30) ? -(1 << 30) : (int)v;
    return 0;
}
/* A window limit as the ABI takes it: 2^30 or more is none. */
static int span_arg(PyObject* o, int* out) {
    if (int_arg(o, out)) return -1;
    if (*out >= (1 << 30)) *out = -1;
    return 0;
}
static int float_arg(PyObject* o, float* out) {
    *out = (float)PyFloat_AsDouble(o);
    return PyErr_Occurred() ? -1 : 0;
}
static int attr_long(PyObject* o, PyObject* name, long long* out) {
    PyObject* v = PyObject_GetAttr(o, name);
    if (!v) return -1;
    *out = PyLong_AsLongLong(v);
    Py_DECREF(v);
    return *out == -1 && PyErr_Occurred() ? -1 : 0;
}

/* A cudasep.KVCache as this file uses it. */
typedef struct {
    const mbr_kv_cache* c;
    PyObject* dtype;
    long long dev;
    PyObject* desc;
} cache_t;
static int cache_arg(PyObject* o, cache_t* x) {
    x->desc = PyObject_GetAttr(o, s_desc);
    if (!x->desc) return -1;
    PyObject* d = PyObject_GetAttr(o, s_cache_dtype);
    if (!d || !PyBytes_Check(x->desc) || PyBytes_GET_SIZE(x->desc) != sizeof(mbr_kv_cache) || attr_long(o, s_dev, &x->dev)) {
        Py_XDECREF(d), Py_DECREF(x->desc);
        if (!PyErr_Occurred()) refuse("expected a KVCache");
        return -1;
    }
    Py_DECREF(d);
    x->dtype = d;
    x->c = (const mbr_kv_cache*)PyBytes_AS_STRING(x->desc);
    return 0;
}

#define NARGS(k)                                                               \
    if (n != (k)) {                                                            \
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");         \
        return NULL;                                                           \
    }

/* qk_norm_rope(q, k, gamma_q, gamma_k, cos, sin, pos, pairs, eps, q_out, k_out, stream) -> (q_out, k_out) */
static PyObject* call_norm(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(12);
    PyObject *q = a[0], *k = a[1], *qo = NULL, *ko = NULL, *res = NULL, *seq = NULL, *dt = NULL;
    rows_t rq, rk, rqo, rko;
    long long dev;
    void *gq, *gk, *c = NULL, *s = NULL, *p = NULL, *st;
    int pairs[8], code, on, axes;
    float eps;
    int64_t tr = 0;
    if (device_of(q, &dev) || !(dt = PyObject_GetAttr(q, s_dtype))) goto done;
    if (rows("q", q, dt, dev, &rq) || rows("k", k, dt, dev, &rk)) goto done;
    if (rk.n[0] != rq.n[0] || rk.n[1] != rq.n[1] || rk.n[3] != rq.n[3]) {
        refuse("q and k must have the same seqs, tokens, dim_head");
        goto done;
    }
    if (!(seq = PySequence_Fast(a[7], "pairs must be a sequence"))) goto done;
    axes = (int)PySequence_Fast_GET_SIZE(seq);
    if (axes > 8) {
        refuse("too many axes");
        goto done;
    }
    for (int i = 0; i < axes; ++i)
        if (int_arg(PySequence_Fast_GET_ITEM(seq, i), &pairs[i])) goto done;
    if (axes) {
        if (a[4] == Py_None || a[5] == Py_None || a[6] == Py_None) {
            refuse("cos, sin and pos are needed with pairs");
            goto done;
        }
        int64_t shape[5];
        if (sizes(a[4], s_shape, 0, shape, 5) < 1) goto done;
        tr = shape[0];
        const int64_t table[2] = {tr, rq.n[3] / 2}, where[3] = {rq.n[0], rq.n[1], axes};
        if (flat("cos", a[4], t_f32, dev, 2, table, &c) || flat("sin", a[5], t_f32, dev, 2, table, &s) ||
            flat("pos", a[6], t_i32, dev, 3, where, &p))
            goto done;
    }
    if (flat("gamma_q", a[2], t_f32, dev, 1, &rq.n[3], &gq) || flat("gamma_k", a[3], t_f32, dev, 1, &rq.n[3], &gk) ||
        float_arg(a[8], &eps) || (code = code_of(dt)) < 0)
        goto done;
    if ((on = stream_of(a[11], dev, &st)) <= 0) {
        if (on == 0) res = elsewhere(dev, "qk_norm_rope", a, n);
        goto done;
    }
    qo = a[9] == Py_None ? like(q, a[11]) : Py_NewRef(a[9]);
    ko = a[10] == Py_None ? like(k, a[11]) : Py_NewRef(a[10]);
    if (!qo || !ko || rows("q_out", qo, dt, dev, &rqo) || rows("k_out", ko, dt, dev, &rko)) goto done;
    for (int i = 0; i < 4; ++i)
        if (rqo.n[i] != rq.n[i] || rko.n[i] != rk.n[i]) {
            refuse("outputs must have the shapes of q and k");
            goto done;
        }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f_norm(&rq.v, &rk.v, &rqo.v, &rko.v, rq.n[0], rq.n[1], (int)rq.n[2], (int)rk.n[2], (int)rq.n[3], gq, gk, eps, c, s,
                tr, p, axes, pairs, code, st);
    Py_END_ALLOW_THREADS;
    if (!checked(rc)) res = PyTuple_Pack(2, qo, ko);
done:
    Py_XDECREF(qo), Py_XDECREF(ko), Py_XDECREF(seq), Py_XDECREF(dt);
    return res;
}

static int same_rows(const rows_t* r, const mbr_kv_cache* c) {
    return r->n[0] == c->seqs && r->n[2] == c->kv_heads && r->n[3] == c->dim_head;
}

/* cache_append(cache, k, v, pos, count, stream) -> None */
static PyObject* call_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(6);
    cache_t x;
    rows_t k, v;
    void *pos, *count, *st;
    PyObject* res = NULL;
    if (cache_arg(a[0], &x)) return NULL;
    if (rows("k", a[1], x.dtype, x.dev, &k) || rows("v", a[2], x.dtype, x.dev, &v)) goto done;
    if (!same_rows(&k, x.c) || !same_rows(&v, x.c) || v.n[1] != k.n[1]) {
        refuse("k and v must be [seqs, tokens, kv_heads, dim_head] of the cache");
        goto done;
    }
    if (a[3] == Py_None) {
        refuse("pos is needed");
        goto done;
    }
    if (flat("pos", a[3], t_i32, x.dev, 1, &k.n[0], &pos) || flat("count", a[4], t_i32, x.dev, 1, &k.n[0], &count)) goto done;
    const int on = stream_of(a[5], x.dev, &st);
    if (on <= 0) {
        if (on == 0) res = elsewhere(x.dev, "cache_append", a, n);
        goto done;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f_append(x.c, &k.v, &v.v, pos, count, k.n[1], st);
    Py_END_ALLOW_THREADS;
    if (!checked(rc)) res = Py_NewRef(Py_None);
done:
    Py_DECREF(x.desc);
    return res;
}

/* cache_read(cache, pos, tokens, count, k, v, stream) -> (k, v) */
static PyObject* call_read(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(7);
    cache_t x;
    rows_t k, v;
    void *pos, *count, *st;
    PyObject *res = NULL, *ko = NULL, *vo = NULL, *shape = NULL;
    if (cache_arg(a[0], &x)) return NULL;
    const long long tokens = PyLong_AsLongLong(a[2]);
    if (tokens == -1 && PyErr_Occurred()) goto done;
    if (tokens < 0) {
        refuse("tokens must not be negative");
        goto done;
    }
    if (a[1] == Py_None) {
        refuse("pos is needed");
        goto done;
    }
    const int64_t seqs = x.c->seqs;
    if (flat("pos", a[1], t_i32, x.dev, 1, &seqs, &pos) || flat("count", a[3], t_i32, x.dev, 1, &seqs, &count)) goto done;
    const int on = stream_of(a[6], x.dev, &st);
    if (on <= 0) {
        if (on == 0) res = elsewhere(x.dev, "cache_read", a, n);
        goto done;
    }
    if (a[4] == Py_None || a[5] == Py_None) {
        shape = Py_BuildValue("(LLii)", (long long)seqs, tokens, x.c->kv_heads, x.c->dim_head);
        if (!shape) goto done;
    }
    ko = a[4] == Py_None ? PyObject_CallMethodObjArgs(a[0], s_new, shape, a[6], NULL) : Py_NewRef(a[4]);
    vo = a[5] == Py_None && ko ? PyObject_CallMethodObjArgs(a[0], s_new, shape, a[6], NULL) : Py_NewRef(a[5]);
    if (!ko || !vo || rows("k", ko, x.dtype, x.dev, &k) || rows("v", vo, x.dtype, x.dev, &v)) goto done;
    if (!same_rows(&k, x.c) || !same_rows(&v, x.c) || k.n[1] != tokens || v.n[1] != tokens) {
        refuse("k and v must be [seqs, tokens, kv_heads, dim_head] of the cache");
        goto done;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f_read(x.c, pos, count, tokens, &k.v, &v.v, st);
    Py_END_ALLOW_THREADS;
    if (!checked(rc)) res = PyTuple_Pack(2, ko, vo);
done:
    Py_DECREF(x.desc), Py_XDECREF(ko), Py_XDECREF(vo), Py_XDECREF(shape);
    return res;
}

/* Workspace of `bytes` for a call on `stream`: the tensor (None for none), or NULL. */
static PyObject* workspace(int64_t bytes, PyObject* t, PyObject* stream, void** ptr) {
    *ptr = NULL;
    if (!bytes) return Py_NewRef(Py_None);
    PyObject* dv = PyObject_GetAttr(t, s_device);
    PyObject* w = dv ? PyObject_CallFunction(p_workspace, "LOO", (long long)bytes, dv, stream) : NULL;
    Py_XDECREF(dv);
    if (w && address(w, ptr)) Py_CLEAR(w);
    return w;
}

/* window_attention(q, k, v, left, right, sinks, scale, q_len, kv_len, gates, out, stream) -> out */
static PyObject* call_window(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(12);
    rows_t q, k, v, o;
    long long dev;
    int left, right, sinks, code, on;
    float scale;
    void *ql, *kl, *g, *st, *wp;
    int64_t bytes = 0;
    PyObject *res = NULL, *out = NULL, *dt = NULL, *work = NULL;
    if (device_of(a[0], &dev) || !(dt = PyObject_GetAttr(a[0], s_dtype))) goto done;
    if (rows("q", a[0], dt, dev, &q) || rows("k", a[1], dt, dev, &k) || rows("v", a[2], dt, dev, &v)) goto done;
    if (k.n[0] != q.n[0] || k.n[3] != q.n[3] || v.n[0] != k.n[0] || v.n[1] != k.n[1] || v.n[2] != k.n[2] || v.n[3] != k.n[3]) {
        refuse("k and v must be [seqs, kv_tokens, kv_heads, dim_head]");
        goto done;
    }
    if (span_arg(a[3], &left) || span_arg(a[4], &right) || int_arg(a[5], &sinks) || float_arg(a[6], &scale) ||
        (code = code_of(dt)) < 0 || flat("q_len", a[7], t_i32, dev, 1, &q.n[0], &ql) ||
        flat("kv_len", a[8], t_i32, dev, 1, &q.n[0], &kl) || flat("gates", a[9], t_f32, dev, 3, q.n, &g))
        goto done;
    if ((on = stream_of(a[11], dev, &st)) <= 0) {
        if (on == 0) res = elsewhere(dev, "window_attention", a, n);
        goto done;
    }
    out = a[10] == Py_None ? like(a[0], a[11]) : Py_NewRef(a[10]);
    if (!out || rows("out", out, dt, dev, &o)) goto done;
    for (int i = 0; i < 4; ++i)
        if (o.n[i] != q.n[i]) {
            refuse("out must have the shape of q");
            goto done;
        }
    if (checked(f_window_ws(q.n[0], q.n[1], k.n[1], (int)q.n[2], (int)k.n[2], (int)q.n[3], left, right, sinks, code, &bytes)) ||
        !(work = workspace(bytes, a[0], a[11], &wp)))
        goto done;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f_window(&q.v, &k.v, &v.v, &o.v, q.n[0], q.n[1], k.n[1], (int)q.n[2], (int)k.n[2], (int)q.n[3], ql, kl, left, right,
                  sinks, scale, g, code, wp, bytes, st);
    Py_END_ALLOW_THREADS;
    if (!checked(rc)) res = Py_NewRef(out);
done:
    Py_XDECREF(out), Py_XDECREF(dt), Py_XDECREF(work);
    return res;
}

/* cache_attention(q, cache, length, left, right, scale, gates, out, stream) -> out */
static PyObject* call_cache(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(9);
    cache_t x;
    rows_t q, o;
    int left, right, on;
    float scale;
    void *len, *g, *st, *wp;
    int64_t bytes = 0;
    PyObject *res = NULL, *out = NULL, *work = NULL;
    if (cache_arg(a[1], &x)) return NULL;
    if (rows("q", a[0], x.dtype, x.dev, &q)) goto done;
    if (q.n[0] != x.c->seqs || q.n[3] != x.c->dim_head) {
        refuse("q must be [seqs, tokens, q_heads, dim_head] of the cache");
        goto done;
    }
    if (a[2] == Py_None) {
        refuse("length is needed");
        goto done;
    }
    if (flat("length", a[2], t_i32, x.dev, 1, &q.n[0], &len) || span_arg(a[3], &left) || span_arg(a[4], &right) ||
        float_arg(a[5], &scale) || flat("gates", a[6], t_f32, x.dev, 3, q.n, &g))
        goto done;
    if ((on = stream_of(a[8], x.dev, &st)) <= 0) {
        if (on == 0) res = elsewhere(x.dev, "cache_attention", a, n);
        goto done;
    }
    out = a[7] == Py_None ? like(a[0], a[8]) : Py_NewRef(a[7]);
    if (!out || rows("out", out, x.dtype, x.dev, &o)) goto done;
    for (int i = 0; i < 4; ++i)
        if (o.n[i] != q.n[i]) {
            refuse("out must have the shape of q");
            goto done;
        }
    if (checked(f_cache_ws(x.c, q.n[1], (int)q.n[2], left, right, &bytes)) || !(work = workspace(bytes, a[0], a[8], &wp)))
        goto done;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f_cache(&q.v, x.c, &o.v, len, q.n[1], (int)q.n[2], left, right, scale, g, wp, bytes, st);
    Py_END_ALLOW_THREADS;
    if (!checked(rc)) res = Py_NewRef(out);
done:
    Py_DECREF(x.desc), Py_XDECREF(out), Py_XDECREF(work);
    return res;
}

/* cache_fields(k, v, k_scale, v_scale, sinks) -> (descriptor, dtype, dev, seqs, kv_heads, dim_head, ring, bits) */
static PyObject* call_fields(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    NARGS(5);
    mbr_kv_cache c;
    int64_t shape[5];
    long long dev;
    int code, sinks;
    PyObject *dt = NULL, *sd = NULL, *res = NULL;
    if (device_of(a[0], &dev) || int_arg(a[4], &sinks) || !(dt = PyObject_GetAttr(a[0], s_dtype))) goto done;
    if (sizes(a[0], s_shape, 0, shape, 5) != 4) {
        if (!PyErr_Occurred()) refuse("k and v must be [seqs, kv_heads, slots, ...]");
        goto done;
    }
    if (a[1] == Py_None) {
        refuse("v is needed");
        goto done;
    }
    if (flat("k", a[0], dt, dev, 4, shape, &c.k) || flat("v", a[1], dt, dev, 4, shape, &c.v)) goto done;
    c.k_scale = c.v_scale = NULL;
    c.bits = 0;
    int64_t dim = shape[3];
    if (dt == t_u8) {
        if (a[2] == Py_None || a[3] == Py_None) {
            refuse("4-bit (uint8) k and v need k_scale and v_scale");
            goto done;
        }
        if (!(sd = PyObject_GetAttr(a[2], s_dtype))) goto done;
        dim = 2 * shape[3];
        c.bits = 4;
        const int64_t ss[5] = {shape[0], shape[1], shape[2], dim / 32, 2};
        if (flat("k_scale", a[2], sd, dev, 5, ss, &c.k_scale) || flat("v_scale", a[3], sd, dev, 5, ss, &c.v_scale)) goto done;
    } else {
        if (a[2] != Py_None || a[3] != Py_None) {
            refuse("k_scale and v_scale go with 4-bit (uint8) k and v");
            goto done;
        }
        sd = Py_NewRef(dt);
    }
    if ((code = code_of(sd)) < 0) goto done;
    if (sinks < 0 || sinks >= shape[2]) {
        refuse("a cache needs slots beyond its sinks");
        goto done;
    }
    if (shape[1] > INT32_MAX || shape[2] > INT32_MAX || dim > INT32_MAX) {
        refuse("kv cache: too large");
        goto done;
    }
    c.seqs = shape[0];
    c.kv_heads = (int)shape[1], c.dim_head = (int)dim, c.sinks = sinks, c.ring = (int)shape[2] - sinks, c.dtype = code;
    res = Py_BuildValue("(y#OLLiiii)", (const char*)&c, (Py_ssize_t)sizeof c, sd, dev, (long long)c.seqs, c.kv_heads,
                        c.dim_head, c.ring, c.bits);
done:
    Py_XDECREF(dt), Py_XDECREF(sd);
    return res;
}

/* bind(addresses, names): the library's entry points and torch's objects. */
static PyObject* call_bind(PyObject* self, PyObject* args) {
    unsigned long long f[7];
    PyObject* o[12];
    if (!PyArg_ParseTuple(args, "(KKKKKKK)(OOOOOOOOOOOO)", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &o[0], &o[1],
                          &o[2], &o[3], &o[4], &o[5], &o[6], &o[7], &o[8], &o[9], &o[10], &o[11]))
        return NULL;
    *(void**)&f_norm = (void*)f[0], *(void**)&f_append = (void*)f[1], *(void**)&f_read = (void*)f[2];
    *(void**)&f_window = (void*)f[3], *(void**)&f_window_ws = (void*)f[4], *(void**)&f_cache = (void*)f[5];
    *(void**)&f_cache_ws = (void*)f[6];
    PyObject** to[12] = {&t_f32,    &t_i32,    &t_u8,    &t_codes,     &p_empty_like, &p_kwargs,
                         &p_stream, &p_device, &p_check, &p_elsewhere, &p_workspace,  &p_like_on};
    for (int i = 0; i < 12; ++i) Py_XSETREF(*to[i], Py_NewRef(o[i]));
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"bind", call_bind, METH_VARARGS, NULL},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))call_norm, METH_FASTCALL, NULL},
    {"cache_fields", (PyCFunction)(void (*)(void))call_fields, METH_FASTCALL, NULL},
    {"cache_append", (PyCFunction)(void (*)(void))call_append, METH_FASTCALL, NULL},
    {"cache_read", (PyCFunction)(void (*)(void))call_read, METH_FASTCALL, NULL},
    {"window_attention", (PyCFunction)(void (*)(void))call_window, METH_FASTCALL, NULL},
    {"cache_attention", (PyCFunction)(void (*)(void))call_cache, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_stream_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__stream_calls(void) {
    struct {
        PyObject** to;
        const char* text;
    } names[] = {{&s_stride, "stride"},         {&s_shape, "shape"},       {&s_dtype, "dtype"},
                 {&s_get_device, "get_device"}, {&s_data_ptr, "data_ptr"}, {&s_contiguous, "is_contiguous"},
                 {&s_device, "device"},         {&s_desc, "_desc"},        {&s_dev, "_dev"},
                 {&s_new, "new"},               {&s_cuda_stream, "cuda_stream"},
                 {&s_cache_dtype, "_dtype"}};
    for (size_t i = 0; i < sizeof names / sizeof *names; ++i)
        if (!(*names[i].to = PyUnicode_InternFromString(names[i].text))) return NULL;
    return PyModule_Create(&module);
}
