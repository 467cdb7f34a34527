/* The hot entry points of libingot_qmm.so as CPython functions. A ctypes call converts every argument through its argtypes
 * object: 2.3 us for iq_qmv, half of what a decode linear of a few megabytes takes on the GPU; through METH_FASTCALL it is
 * 0.3 us. Arguments are integers (addresses, sizes, flags) and, where the C signature has them, floats, or (the last three entries) tensors; the
 * result is the status. The library is already loaded (capi.lib()); bind(name, address) hands over the symbols. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <string.h>

#include "../../include/ingot_qmm.h"

static void* fn_qmv;
static void* fn_qmm;
static void* fn_dense_ffn;
static void* fn_moe_forward;
static void* fn_rmsnorm;
static void* fn_had_rows;
static void* fn_embed_rows;
static void* fn_argmax_rows;
static void* fn_topk64;
static void* fn_add_rmsnorm;
static void* fn_qmm_i8;
static void* fn_logits_rules;

static const struct { const char* name; void** slot; } table[] = {
    {"iq_qmv", &fn_qmv},           {"iq_qmm", &fn_qmm},               {"iq_dense_ffn", &fn_dense_ffn},
    {"iq_moe_forward", &fn_moe_forward}, {"iq_rmsnorm", &fn_rmsnorm}, {"iq_had_rows", &fn_had_rows},
    {"iq_embed_rows", &fn_embed_rows},   {"iq_argmax_rows", &fn_argmax_rows}, {"iq_topk64", &fn_topk64},
    {"iq_add_rmsnorm", &fn_add_rmsnorm}, {"iq_qmm_i8", &fn_qmm_i8}, {"iq_logits_rules", &fn_logits_rules},
};

static PyObject* py_bind(PyObject* self, PyObject* args) {
    const char* name;
    unsigned long long addr;
    (void)self;
    if (!PyArg_ParseTuple(args, "sK", &name, &addr)) return NULL;
    for (size_t i = 0; i < sizeof(table) / sizeof(table[0]); i++)
        if (strcmp(table[i].name, name) == 0) {
            *table[i].slot = (void*)(uintptr_t)addr;
            Py_RETURN_NONE;
        }
    PyErr_Format(PyExc_KeyError, "no entry point %s", name);
    return NULL;
}

/* argument i as a 64-bit pattern; a conversion error is looked for once, after all of them */
static inline uint64_t U(PyObject* const* a, int i) {
    if (a[i] == Py_None) return 0;
    return PyLong_AsUnsignedLongLongMask(a[i]);
}
#define P(i) ((void*)(uintptr_t)U(a, i))
#define I32(i) ((int32_t)U(a, i))
#define I64(i) ((int64_t)U(a, i))
#define U32(i) ((uint32_t)U(a, i))
#define F32(i) ((float)PyFloat_AsDouble(a[i]))

#define ENTRY(NAME, COUNT, TYPE, ...)                                                                \
    static PyObject* py_##NAME(PyObject* self, PyObject* const* a, Py_ssize_t n) {                  \
        (void)self;                                                                                 \
        if (n != COUNT || fn_##NAME == NULL) {                                                      \
            PyErr_SetString(PyExc_TypeError, #NAME ": wrong number of arguments, or not bound");    \
            return NULL;                                                                            \
        }                                                                                           \
        TYPE f = (TYPE)fn_##NAME;                                                                   \
        int32_t st;                                                                                 \
        __VA_ARGS__;                                                                                 \
        return PyLong_FromLong(st);                                                                 \
    }
/* converts every argument first, so that nothing is launched when one of them is not a number */
#define CHECKED if (PyErr_Occurred()) return NULL
/* a launch can block on a full queue: other threads run meanwhile */
#define LAUNCH(CALL_) Py_BEGIN_ALLOW_THREADS st = CALL_; Py_END_ALLOW_THREADS

typedef int32_t (*qmv_t)(iq_ctx*, void*, const void*, int32_t, int64_t, const iq_qlinear*, void*, int32_t, int64_t, int32_t,
                         uint32_t, int32_t);
ENTRY(qmv, 12, qmv_t, {
    void *c = P(0), *s = P(1), *x = P(2), *q = P(5), *y = P(6);
    int32_t xd = I32(3), yd = I32(7), rows = I32(9), np = I32(11);
    int64_t ldx = I64(4), ldy = I64(8);
    uint32_t fl = U32(10);
    CHECKED;
    LAUNCH(f(c, s, x, xd, ldx, q, y, yd, ldy, rows, fl, np));
})
typedef int32_t (*qmm_t)(iq_ctx*, void*, const void*, int32_t, int64_t, const iq_qlinear*, void*, int32_t, int64_t, int32_t,
                         uint32_t, void*, size_t);
ENTRY(qmm, 13, qmm_t, {
    void *c = P(0), *s = P(1), *x = P(2), *q = P(5), *y = P(6), *ws = P(11);
    int32_t xd = I32(3), yd = I32(7), rows = I32(9);
    int64_t ldx = I64(4), ldy = I64(8);
    uint32_t fl = U32(10);
    size_t wb = (size_t)U(a, 12);
    CHECKED;
    LAUNCH(f(c, s, x, xd, ldx, q, y, yd, ldy, rows, fl, ws, wb));
})
typedef int32_t (*ffn_t)(iq_ctx*, void*, const void*, int32_t, int64_t, const iq_qlinear*, const iq_qlinear*, int32_t, float,
                         void*, int32_t, int64_t, int32_t, uint32_t, void*, size_t);
ENTRY(dense_ffn, 16, ffn_t, {
    void *c = P(0), *s = P(1), *x = P(2), *g = P(5), *d = P(6), *o = P(9), *ws = P(14);
    int32_t xd = I32(3), act = I32(7), od = I32(10), rows = I32(12);
    int64_t ldx = I64(4), ldo = I64(11);
    float lim = F32(8);
    uint32_t fl = U32(13);
    size_t wb = (size_t)U(a, 15);
    CHECKED;
    LAUNCH(f(c, s, x, xd, ldx, g, d, act, lim, o, od, ldo, rows, fl, ws, wb));
})
typedef int32_t (*moe_t)(iq_moe*, void*, const void*, int32_t, int64_t, void*, int32_t, int64_t, int32_t, uint32_t, uint32_t, void*,
                         size_t);
ENTRY(moe_forward, 13, moe_t, {
    void *l = P(0), *s = P(1), *x = P(2), *o = P(5), *ws = P(11);
    int32_t xd = I32(3), od = I32(6), rows = I32(8);
    int64_t ldx = I64(4), ldo = I64(7);
    uint32_t fl = U32(9), pieces = U32(10);
    size_t wb = (size_t)U(a, 12);
    CHECKED;
    LAUNCH(f(l, s, x, xd, ldx, o, od, ldo, rows, fl, pieces, ws, wb));
})
typedef int32_t (*norm_t)(iq_ctx*, void*, const float*, int64_t, void*, int32_t, int64_t, int32_t, int32_t, float);
ENTRY(rmsnorm, 10, norm_t, {
    void *c = P(0), *s = P(1), *x = P(2), *o = P(4);
    int64_t ldx = I64(3), ldo = I64(6);
    int32_t od = I32(5), rows = I32(7), d = I32(8);
    float eps = F32(9);
    CHECKED;
    LAUNCH(f(c, s, x, ldx, o, od, ldo, rows, d, eps));
})
typedef int32_t (*had_t)(iq_ctx*, void*, const void*, int32_t, int64_t, const float*, void*, int64_t, int32_t, int32_t);
ENTRY(had_rows, 10, had_t, {
    void *c = P(0), *s = P(1), *x = P(2), *sg = P(5), *y = P(6);
    int32_t xd = I32(3), rows = I32(8), k = I32(9);
    int64_t ldx = I64(4), ldy = I64(7);
    CHECKED;
    LAUNCH(f(c, s, x, xd, ldx, sg, y, ldy, rows, k));
})
typedef int32_t (*embed_t)(iq_ctx*, void*, const iq_qlinear*, const uint32_t*, int32_t, float*, void*, int64_t);
ENTRY(embed_rows, 8, embed_t, {
    void *c = P(0), *s = P(1), *q = P(2), *tok = P(3), *of = P(5), *oh = P(6);
    int32_t rows = I32(4);
    int64_t ldo = I64(7);
    CHECKED;
    LAUNCH(f(c, s, q, tok, rows, of, oh, ldo));
})
typedef int32_t (*argmax_t)(iq_ctx*, void*, const float*, int64_t, int32_t, int32_t, uint32_t*);
ENTRY(argmax_rows, 7, argmax_t, {
    void *c = P(0), *s = P(1), *x = P(2), *o = P(6);
    int64_t ldx = I64(3);
    int32_t rows = I32(4), nn = I32(5);
    CHECKED;
    LAUNCH(f(c, s, x, ldx, rows, nn, o));
})
typedef int32_t (*topk_t)(iq_ctx*, void*, const float*, int64_t, int32_t, int32_t, const float*, int32_t, uint32_t*, float*, float*,
                          void*, size_t);
ENTRY(topk64, 13, topk_t, {
    void *c = P(0), *s = P(1), *x = P(2), *t = P(6), *ix = P(8), *v = P(9), *z = P(10), *sc = P(11);
    int64_t ldx = I64(3);
    int32_t rows = I32(4), vocab = I32(5), nt = I32(7);
    size_t sb = (size_t)U(a, 12);
    CHECKED;
    LAUNCH(f(c, s, x, ldx, rows, vocab, t, nt, ix, v, z, sc, sb));
})

/* ---- entry points that take the tensors themselves ----------------------------------------------------------------------------
 * What a tensor says of itself is asked for here: from Python its shape, strides, type, device and address and the conditions on them cost as much as
 * the launch. A tensor that is not as the entry wants it makes the result None, before anything is launched; the caller then says why. */
static PyObject *s_shape, *s_stride, *s_dtype, *s_get_device, *s_data_ptr, *s_numel, *s_is_contiguous;
static PyObject* types[4]; /* float32, float16, bfloat16 in the order of iq_dtype, int8 */

typedef struct {
    void* p;
    int64_t rows, cols, ld; /* [rows, cols], rows ld elements apart; one dimension: [rows] */
    int type;               /* index in types, -1: none of them */
} Rows;

static int number(PyObject* o, int64_t* v) {
    if (o == NULL) return -1;
    *v = (int64_t)PyLong_AsUnsignedLongLongMask(o);
    Py_DECREF(o);
    return PyErr_Occurred() ? -1 : 0;
}
static int type_of(PyObject* t) {
    PyObject* d = PyObject_GetAttr(t, s_dtype);
    int i = 3;
    if (d == NULL) return -1;
    while (i >= 0 && types[i] != d) i--;
    Py_DECREF(d);
    return i;
}
/* A tensor of `dims` (one or two) dimensions on the device, of two with neighbouring elements in a row. 0: o is filled. */
static int rows_of(PyObject* t, int dims, int64_t device, Rows* o) {
    int64_t dev, addr, size[2] = {0, 0}, step[2] = {0, 0};
    PyObject *shape = PyObject_GetAttr(t, s_shape), *stride = NULL;
    int ok = 0;
    if (shape == NULL || !PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != dims) goto out;
    stride = PyObject_CallMethodNoArgs(t, s_stride);
    if (stride == NULL || !PyTuple_Check(stride) || PyTuple_GET_SIZE(stride) != dims) goto out;
    for (int i = 0; i < dims; i++) {
        size[i] = (int64_t)PyLong_AsUnsignedLongLongMask(PyTuple_GET_ITEM(shape, i));
        step[i] = (int64_t)PyLong_AsUnsignedLongLongMask(PyTuple_GET_ITEM(stride, i));
    }
    if (PyErr_Occurred() || number(PyObject_CallMethodNoArgs(t, s_get_device), &dev) || dev != device || number(PyObject_CallMethodNoArgs(t, s_data_ptr), &addr)) goto out;
    if (dims == 2 && step[1] != 1 && size[1] > 1) goto out;
    o->p = (void*)(uintptr_t)addr;
    o->rows = size[0];
    o->cols = dims == 2 ? size[1] : 1;
    o->ld = step[0];
    o->type = type_of(t);
    ok = 1;
out:
    Py_XDECREF(shape);
    Py_XDECREF(stride);
    return ok ? 0 : -1;
}
static PyObject* not_taken(void) {
    PyErr_Clear();
    Py_RETURN_NONE;
}
#define TENSORS(NAME, COUNT)                                                                    \
    if (n != COUNT || fn_##NAME == NULL || types[0] == NULL) {                                  \
        PyErr_SetString(PyExc_TypeError, #NAME ": wrong number of arguments, or not bound");    \
        return NULL;                                                                            \
    }
#define FLOATS(T) ((T).type >= 0 && (T).type <= 2)

static PyObject* py_bind_types(PyObject* self, PyObject* args) {
    PyObject* t[4];
    (void)self;
    if (!PyArg_ParseTuple(args, "OOOO", &t[0], &t[1], &t[2], &t[3])) return NULL;
    for (int i = 0; i < 4; i++) {
        Py_INCREF(t[i]);
        types[i] = t[i];
    }
    Py_RETURN_NONE;
}

typedef int32_t (*add_norm_t)(iq_ctx*, void*, const void*, int32_t, int64_t, const void*, int32_t, int64_t, void*, int64_t, const void*, int32_t,
                              float, float, int32_t, int32_t, void*, int32_t, int64_t, int8_t*, int64_t, float*, int32_t);
/* (context, stream, device, x, residual, weight, rows, eps, weight_offset, residual_out, out, codes, scales, rotate) */
static PyObject* py_add_rmsnorm(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    TENSORS(add_rmsnorm, 14);
    (void)self;
    void *c = P(0), *s = P(1), *w = NULL;
    const int64_t device = I64(2), rows = I64(6), rotate = I64(13);
    const double eps = PyFloat_AsDouble(a[7]), offset = PyFloat_AsDouble(a[8]);
    Rows x = {0}, r, ro = {0}, o = {0}, q = {0}, sc = {0};
    int wd = 0;
    if (PyErr_Occurred()) return not_taken();
    if (rows_of(a[4], 2, device, &r) || !FLOATS(r) || rows < 0 || r.rows < rows || r.cols < 1 || r.cols > 32768 || !(eps >= 0)) return not_taken();
#define LIKE(T) ((T).rows >= rows && (T).cols == r.cols)
    if (a[3] != Py_None) {
        if (rows_of(a[3], 2, device, &x) || !FLOATS(x) || !LIKE(x)) return not_taken();
        ro = r;
        if (a[9] != Py_None && (rows_of(a[9], 2, device, &ro) || ro.type != r.type || !LIKE(ro))) return not_taken();
    } else if (a[9] != Py_None) {
        return not_taken();
    }
    if (a[5] != Py_None) {
        int64_t dev, numel, addr;
        PyObject* whole = PyObject_CallMethodNoArgs(a[5], s_is_contiguous);
        Py_XDECREF(whole);
        wd = type_of(a[5]);
        if (whole != Py_True || wd < 0 || wd > 2 || number(PyObject_CallMethodNoArgs(a[5], s_get_device), &dev) || dev != device ||
            number(PyObject_CallMethodNoArgs(a[5], s_numel), &numel) || numel != r.cols || number(PyObject_CallMethodNoArgs(a[5], s_data_ptr), &addr))
            return not_taken();
        w = (void*)(uintptr_t)addr;
    }
    if (a[10] != Py_None && (rows_of(a[10], 2, device, &o) || !FLOATS(o) || !LIKE(o))) return not_taken();
    if (a[11] != Py_None) {
        if (rows_of(a[11], 2, device, &q) || q.type != 3 || !LIKE(q) || rows_of(a[12], 1, device, &sc) || sc.type != 0 || sc.rows < rows || (rows > 1 && sc.ld != 1)) return not_taken();
    } else if (a[12] != Py_None) {
        return not_taken();
    }
#undef LIKE
    if ((rotate != 0 && rotate != 32 && rotate != 256) || (rotate != 0 && (a[11] == Py_None || r.cols % rotate != 0)) || (a[10] == Py_None && a[11] == Py_None) ||
        rows > INT32_MAX)
        return not_taken();
    if (rows == 0) return PyLong_FromLong(0); /* (tensors of no rows have no address) */
    if (rows == 1) x.ld = r.ld = ro.ld = o.ld = q.ld = r.cols; /* (one row has no stride) */
    const add_norm_t f = (add_norm_t)fn_add_rmsnorm;
    int32_t st;
    LAUNCH(f(c, s, x.p, x.type, x.ld, r.p, r.type, r.ld, ro.p, ro.ld, w, wd, (float)offset, (float)eps, (int32_t)rows, (int32_t)r.cols, o.p, o.type, o.ld, q.p, q.ld, sc.p,
             (int32_t)rotate));
    return PyLong_FromLong(st);
}

typedef int32_t (*qmm_i8_t)(iq_ctx*, void*, const int8_t*, int64_t, const float*, const int8_t*, const float*, int32_t, int32_t, void*, int32_t, int64_t,
                            int32_t, uint32_t);
/* (context, stream, device, x, x_scales, address of w, address of w_scales, n, k, y, rows, flags) */
static PyObject* py_qmm_i8(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    TENSORS(qmm_i8, 12);
    (void)self;
    void *c = P(0), *s = P(1), *w = P(5), *sw = P(6);
    const int64_t device = I64(2), nn = I64(7), k = I64(8), rows = I64(10);
    const uint32_t flags = U32(11);
    Rows x, sx, y;
    if (PyErr_Occurred()) return not_taken();
    if (rows_of(a[3], 2, device, &x) || x.type != 3 || x.cols != k || rows < 0 || rows > INT32_MAX || x.rows < rows || rows_of(a[4], 1, device, &sx) || sx.type != 0 ||
        sx.rows < rows || (rows > 1 && sx.ld != 1) || rows_of(a[9], 2, device, &y) || !FLOATS(y) || y.cols != nn || y.rows < rows)
        return not_taken();
    if (rows == 0) return PyLong_FromLong(0);
    if (rows == 1) x.ld = k, y.ld = nn;
    const qmm_i8_t f = (qmm_i8_t)fn_qmm_i8;
    int32_t st;
    LAUNCH(f(c, s, x.p, x.ld, sx.p, w, sw, (int32_t)nn, (int32_t)k, y.p, y.type, y.ld, (int32_t)rows, flags));
    return PyLong_FromLong(st);
}

typedef int32_t (*rules_t)(iq_ctx*, void*, const void*, int32_t, int64_t, float*, int64_t, int32_t, int32_t, const iq_logit_rules*);
/* (context, stream, device, x, out, rows, vocab, address of the rules) */
static PyObject* py_logits_rules(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    TENSORS(logits_rules, 8);
    (void)self;
    void *c = P(0), *s = P(1), *rules = P(7);
    const int64_t device = I64(2), rows = I64(5), vocab = I64(6);
    Rows x, o;
    if (PyErr_Occurred()) return not_taken();
    if (rows_of(a[3], 2, device, &x) || !FLOATS(x) || x.cols != vocab || rows < 0 || rows > INT32_MAX || x.rows < rows || rows_of(a[4], 2, device, &o) || o.type != 0 ||
        o.cols != vocab || o.rows < rows)
        return not_taken();
    if (rows == 0) return PyLong_FromLong(0);
    if (rows == 1) x.ld = o.ld = vocab;
    const rules_t f = (rules_t)fn_logits_rules;
    int32_t st;
    LAUNCH(f(c, s, x.p, x.type, x.ld, o.p, o.ld, (int32_t)rows, (int32_t)vocab, rules));
    return PyLong_FromLong(st);
}

#define M(NAME) {#NAME, (PyCFunction)(void (*)(void))py_##NAME, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, NULL}, {"bind_types", py_bind_types, METH_VARARGS, NULL}, M(qmv), M(qmm), M(dense_ffn), M(moe_forward), M(rmsnorm), M(had_rows), M(embed_rows),
    M(argmax_rows), M(topk64), M(add_rmsnorm), M(qmm_i8), M(logits_rules), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_iqcall", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__iqcall(void) {
    static const struct { PyObject** slot; const char* name; } names[] = {{&s_shape, "shape"}, {&s_stride, "stride"}, {&s_dtype, "dtype"}, {&s_get_device, "get_device"},
                                                                         {&s_data_ptr, "data_ptr"}, {&s_numel, "numel"}, {&s_is_contiguous, "is_contiguous"}};
    for (size_t i = 0; i < sizeof(names) / sizeof(names[0]); i++)
        if ((*names[i].slot = PyUnicode_InternFromString(names[i].name)) == NULL) return NULL;
    return PyModule_Create(&module);
}
