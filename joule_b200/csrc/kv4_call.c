/* The regular calls of joule_b200/kv4.py without the interpreter's and ctypes' share
 * of their time (a call on a short cache took 10 us of the host, 2.6 of them the
 * launch). Each function checks what the Python function checks and, when all of it
 * holds and the tensors lie as the library takes them (contiguous, on the current
 * device), makes the call; otherwise it returns None and has done nothing, and the
 * Python function goes on: it copies, changes streams, or raises. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <math.h>

#include "joule_moe.h"

static PyObject *n_shape, *n_dtype, *n_data_ptr, *n_is_contiguous, *n_get_device, *n_new_empty, *kw_dtype;
/* set by bind(): torch's dtypes and functions, the library's entry points */
static PyObject *t_u8, *t_i32, *t_types[3], *f_empty_like, *f_device, *f_stream;
static int (*p_append)(const jl_kv4*, int, const void*, const void*, int, long long, long long, const int*, const int*,
                       int, int*, void*);
static int (*p_read)(const jl_kv4*, int, const int*, const int*, int, void*, void*, int, int*, void*);
static int (*p_attn)(const jl_kv4*, int, const void*, int, long long, const int*, const int*, int, int, int, int, float,
                     void*, void*, long long, int*, void*);
static long long (*p_ws)(const jl_kv4*, int, int, int, int);

/* What of a tensor the calls need; 0 when it is not regular or not a tensor. */
typedef struct {
    long long dim[5];
    int dims, dev;
    PyObject* dtype; /* a singleton: only compared */
    char* p;
} view;

static int int_of(PyObject* o, long long* x) {
    if (!o) return 0;
    *x = PyLong_AsLongLong(o);
    Py_DECREF(o);
    return !(*x == -1 && PyErr_Occurred());
}

static PyObject* method(PyObject* o, PyObject* name) { return PyObject_CallMethodNoArgs(o, name); }

static int look(PyObject* t, view* v) {
    long long x;
    PyObject* o = PyObject_GetAttr(t, n_shape);
    if (!o) return 0;
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) > 5) {
        Py_DECREF(o);
        return 0;
    }
    v->dims = (int)PyTuple_GET_SIZE(o);
    for (int i = 0; i < v->dims; i++) {
        v->dim[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
        if (v->dim[i] < 0) {
            Py_DECREF(o);
            return 0;
        }
    }
    Py_DECREF(o);
    if (!(v->dtype = PyObject_GetAttr(t, n_dtype))) return 0;
    Py_DECREF(v->dtype); /* torch's module holds it */
    if (!(o = method(t, n_is_contiguous))) return 0;
    Py_DECREF(o);
    if (o != Py_True) return 0;
    if (!int_of(method(t, n_get_device), &x) || x < 0) return 0;
    v->dev = (int)x;
    if (!int_of(method(t, n_data_ptr), &x)) return 0;
    v->p = (char*)(uintptr_t)x;
    return 1;
}

static int kind_of(PyObject* dtype) {
    for (int i = 0; i < 3; i++)
        if (dtype == t_types[i]) return i;
    return -1;
}

/* The cache, the layer, and that the cache's device is the current one; its stream. */
static int look_cache(PyObject* cache, PyObject* layer, jl_kv4* c, int* l, int* dev, void** stream) {
    view v;
    long long x;
    if (!look(cache, &v) || v.dims != 5 || v.dtype != t_u8 || !PyLong_Check(layer)) return 0;
    for (int i = 0; i < 4; i++)
        if (v.dim[i] < 1 || v.dim[i] > INT_MAX) return 0;
    if ((v.dim[4] != 68 * 64 && v.dim[4] != 68 * 128) || v.dim[3] > INT_MAX / 64) return 0;
    x = PyLong_AsLongLong(layer);
    if (x < 0 || x >= v.dim[1]) return 0;
    *l = (int)x;
    c->base = v.p, c->slots = (int)v.dim[0], c->L = (int)v.dim[1], c->n_kv = (int)v.dim[2], c->hd = (int)v.dim[4] / 68;
    c->maxT = (int)v.dim[3] * 64;
    *dev = v.dev;
    if (!int_of(PyObject_CallNoArgs(f_device), &x) || x != v.dev) return 0;
    PyObject* d = PyLong_FromLong(v.dev);
    const int ok = d && int_of(PyObject_CallOneArg(f_stream, d), &x);
    Py_XDECREF(d);
    *stream = (void*)(uintptr_t)x;
    return ok;
}

/* A contiguous int32 tensor of n on the device. */
static const int* look_index(PyObject* t, long long n, int dev) {
    view v;
    if (!look(t, &v) || v.dims != 1 || v.dim[0] != n || v.dtype != t_i32 || v.dev != dev) return NULL;
    return (const int*)v.p;
}

/* No answer: the Python function goes on (an error in looking at something is its to raise). */
static PyObject* pass(void) {
    PyErr_Clear();
    Py_RETURN_NONE;
}

/* append(cache, l, k, v, slots, positions): the library's code. */
static PyObject* append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    jl_kv4 c;
    view k, v;
    int l, dev, kind, rc;
    void* stream;
    const int *s, *p;
    if (n != 6 || !look_cache(a[0], a[1], &c, &l, &dev, &stream) || !look(a[2], &k) || !look(a[3], &v)) return pass();
    if (k.dims != 3 || v.dims != 3 || k.dim[0] < 1 || k.dim[0] > INT_MAX || v.dim[0] != k.dim[0] || k.dim[1] != c.n_kv ||
        v.dim[1] != c.n_kv || k.dim[2] != c.hd || v.dim[2] != c.hd || k.dtype != v.dtype || (kind = kind_of(k.dtype)) < 0 ||
        k.dev != dev || v.dev != dev || (uintptr_t)k.p % 16 || (uintptr_t)v.p % 16)
        return pass();
    if (!(s = look_index(a[4], k.dim[0], dev)) || !(p = look_index(a[5], k.dim[0], dev))) return pass();
    const long long row = (long long)c.n_kv * c.hd;
    Py_BEGIN_ALLOW_THREADS;
    rc = p_append(&c, l, k.p, v.p, kind, row, row, s, p, (int)k.dim[0], NULL, stream);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(rc);
}

/* A tensor on the cache's device (half a microsecond less than torch.empty). */
static PyObject* empty(PyObject* cache, PyObject* shape, PyObject* dtype) {
    PyObject* args[3] = {cache, shape, dtype};
    return PyObject_VectorcallMethod(n_new_empty, args, 2, kw_dtype);
}

/* read(cache, l, slots, positions, dtype): (code, k, v). */
static PyObject* read_back(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    jl_kv4 c;
    view s;
    int l, dev, kind, rc = 0;
    void* stream;
    const int* p;
    if (n != 5 || (kind = kind_of(a[4])) < 0 || !look_cache(a[0], a[1], &c, &l, &dev, &stream) || !look(a[2], &s)) return pass();
    if (s.dims != 1 || s.dim[0] < 1 || s.dim[0] > INT_MAX || s.dtype != t_i32 || s.dev != dev ||
        !(p = look_index(a[3], s.dim[0], dev)))
        return pass();
    PyObject *shape = Py_BuildValue("(Lii)", s.dim[0], c.n_kv, c.hd), *k = NULL, *v = NULL, *r = NULL;
    long long pk, pv;
    if (shape && (k = empty(a[0], shape, a[4])) && (v = PyObject_CallOneArg(f_empty_like, k)) &&
        int_of(method(k, n_data_ptr), &pk) && int_of(method(v, n_data_ptr), &pv)) {
        Py_BEGIN_ALLOW_THREADS;
        rc = p_read(&c, l, (const int*)s.p, p, (int)s.dim[0], (void*)(uintptr_t)pk, (void*)(uintptr_t)pv, kind, NULL, stream);
        Py_END_ALLOW_THREADS;
        r = Py_BuildValue("(iOO)", rc, k, v);
    }
    Py_XDECREF(shape), Py_XDECREF(k), Py_XDECREF(v);
    return r; /* NULL: allocation raised */
}

/* attention(cache, l, q, slots, lens, scale or None, longest or None): (code, out). */
static PyObject* attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    jl_kv4 c;
    view q;
    int l, dev, kind, rc = 0;
    void* stream;
    const int *s, *p;
    if (n != 7 || !look_cache(a[0], a[1], &c, &l, &dev, &stream) || !look(a[2], &q)) return pass();
    if (q.dims != 3 && q.dims != 4) return pass();
    const long long B = q.dim[0], T = q.dims == 4 ? q.dim[1] : 1, H = q.dim[q.dims - 2];
    if (q.dim[q.dims - 1] != c.hd || B < 1 || B > INT_MAX || T < 1 || T > INT_MAX || H < 1 || H > INT_MAX || H % c.n_kv ||
        (kind = kind_of(q.dtype)) < 0 || q.dev != dev || (uintptr_t)q.p % 16)
        return pass();
    if (!(s = look_index(a[3], B, dev)) || !(p = look_index(a[4], B, dev))) return pass();
    const double scale = a[5] == Py_None ? 1.0 / sqrt((double)c.hd) : PyFloat_AsDouble(a[5]);
    long long longest = 0;
    if (a[6] != Py_None && (!PyLong_Check(a[6]) || (longest = PyLong_AsLongLong(a[6])) < 1 || longest > c.maxT)) return pass();
    if (PyErr_Occurred()) return pass();
    const long long need = p_ws(&c, (int)B, (int)T, (int)H, (int)longest);
    PyObject *out = PyObject_CallOneArg(f_empty_like, a[2]), *ws = NULL, *r = NULL;
    long long po = 0, pw = 0;
    if (out && need > 0) {
        PyObject* size = PyLong_FromLongLong(need);
        if (size) ws = empty(a[0], size, t_u8);
        Py_XDECREF(size);
    }
    if (out && (need <= 0 || (ws && int_of(method(ws, n_data_ptr), &pw))) && int_of(method(out, n_data_ptr), &po)) {
        Py_BEGIN_ALLOW_THREADS;
        rc = p_attn(&c, l, q.p, kind, H * c.hd, s, p, (int)longest, (int)B, (int)T, (int)H, (float)scale, (void*)(uintptr_t)po,
                    (void*)(uintptr_t)pw, need > 0 ? need : 0, NULL, stream);
        Py_END_ALLOW_THREADS;
        r = Py_BuildValue("(iO)", rc, out);
    }
    Py_XDECREF(out), Py_XDECREF(ws);
    return r;
}

/* bind(uint8, int32, fp32, fp16, bf16, empty_like, current_device, current_stream, append, read, attn, ws) */
static PyObject* bind(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    PyObject** keep[8] = {&t_u8, &t_i32, &t_types[JL_F32], &t_types[JL_F16], &t_types[JL_BF16], &f_empty_like, &f_device, &f_stream};
    if (n != 12) {
        PyErr_SetString(PyExc_TypeError, "bind takes 12 arguments");
        return NULL;
    }
    void* at[4];
    for (int i = 0; i < 4; i++)
        if (!(at[i] = PyLong_AsVoidPtr(a[8 + i]))) return PyErr_Occurred() ? NULL : pass();
    p_append = at[0], p_read = at[1], p_attn = at[2], p_ws = at[3];
    for (int i = 0; i < 8; i++) {
        Py_INCREF(a[i]);
        Py_XSETREF(*keep[i], a[i]);
    }
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, NULL},
                                {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, NULL},
                                {"read", (PyCFunction)(void (*)(void))read_back, METH_FASTCALL, NULL},
                                {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4_call", "Regular calls of joule_b200.kv4.", -1, methods};

PyMODINIT_FUNC PyInit__kv4_call(void) {
    n_shape = PyUnicode_InternFromString("shape");
    n_dtype = PyUnicode_InternFromString("dtype");
    n_data_ptr = PyUnicode_InternFromString("data_ptr");
    n_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    n_get_device = PyUnicode_InternFromString("get_device");
    n_new_empty = PyUnicode_InternFromString("new_empty");
    kw_dtype = Py_BuildValue("(s)", "dtype");
    if (!n_shape || !n_dtype || !n_data_ptr || !n_is_contiguous || !n_get_device || !n_new_empty || !kw_dtype) return NULL;
    return PyModule_Create(&module);
}
