/* berth_b200._bind: the callers of the operators that take shapes and strides from torch tensors (rope, logprobs, route), in C.
 * A decode step calls them with a few rows at a time, and reading eight tensors and checking them in Python took longer (6 us of
 * 10) than the kernels.  No torch headers: a tensor is read through the C function that torch.Tensor publishes for this (DLPack's
 * exchange interface, version 1; asking eight tensors for five attributes each took 2 us).  Every check is made before the library
 * is called; the library's error becomes berth_b200.kernels.Error, set by init(). */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>

#include "../../include/berth_b200.h"

/* DLPack 1.x, the parts in use */
typedef struct { uint32_t major, minor; } dl_version;
typedef struct {
    void* data;
    int32_t device_type, device_id;
    int32_t ndim;
    struct { uint8_t code, bits; uint16_t lanes; } dtype;
    int64_t *shape, *strides;
    uint64_t byte_offset;
} dl_tensor;
typedef struct {
    dl_version version;
    void *previous, *allocate, *managed_from_object, *managed_to_object;
    int (*tensor_from_object)(void* object, dl_tensor* out);   /* borrowed from the object */
    void* current_stream;
} dl_exchange;
enum { DL_CUDA = 2 };

/* types: DLPack's code (0 integer, 2 float, 4 bfloat) and bits */
enum { T_INT32 = 0 << 8 | 32, T_HALF = 2 << 8 | 16, T_FLOAT = 2 << 8 | 32, T_DOUBLE = 2 << 8 | 64, T_BFLOAT16 = 4 << 8 | 16 };

static PyObject* g_error;
static PyTypeObject* g_tensor;
static const dl_exchange* g_exchange;

typedef struct {
    int given;           /* not None */
    int dev, dtype;
    void* ptr;
    int64_t shape[3], stride[3];
} tensor;

static int fail(const char* what, const char* name, const char* msg)
{
    PyErr_Format(g_error, "%s: %s %s", what, name, msg);
    return -1;
}

/* A tensor of nd dimensions with contiguous innermost elements, or None where it may be. */
static int read_tensor(PyObject* o, const char* what, const char* name, int nd, int optional, tensor* t)
{
    t->given = o != Py_None;
    t->ptr = NULL;
    t->dtype = -1;
    if (!t->given) return optional ? 0 : fail(what, name, "is missing");
    if (!PyObject_TypeCheck(o, g_tensor)) return fail(what, name, "must be a torch tensor");
    dl_tensor d;
    if (g_exchange->tensor_from_object(o, &d)) {
        PyErr_Clear();
        return fail(what, name, "must be a dense torch tensor");
    }
    if (d.ndim != nd) {
        PyErr_Format(g_error, "%s: %s must have %d dimensions, got %d", what, name, nd, (int) d.ndim);
        return -1;
    }
    if (d.device_type != DL_CUDA) return fail(what, name, "must be on the CUDA device");
    t->dev = d.device_id;
    t->dtype = d.dtype.lanes == 1 ? d.dtype.code << 8 | d.dtype.bits : -1;
    t->ptr = (char*) d.data + d.byte_offset;
    for (int i = 0; i < nd; ++i) {
        t->shape[i] = d.shape[i];
        t->stride[i] = d.strides[i];
    }
    if (t->shape[nd - 1] > 1 && t->stride[nd - 1] != 1) return fail(what, name, "must have contiguous innermost elements");
    return 0;
}

static const char* type_name(int dtype)
{
    switch (dtype) {
        case T_INT32: return "int32";
        case T_FLOAT: return "float32";
        default: return "bfloat16";   /* (what read_flat is asked for) */
    }
}

/* A contiguous tensor of the given type and shape (nd 1 or 2), or None. */
static int read_flat(PyObject* o, const char* what, const char* name, int dtype, int nd, int64_t rows, int64_t cols, tensor* t)
{
    if (read_tensor(o, what, name, nd, 1, t)) return -1;
    if (!t->given) return 0;
    if (t->dtype != dtype || t->shape[0] != rows || (nd == 2 && (t->shape[1] != cols || (rows > 1 && cols > 0 && t->stride[0] != cols)))) {
        if (nd == 1) PyErr_Format(g_error, "%s: %s must be a contiguous %s tensor of shape (%lld,)", what, name, type_name(dtype), (long long) rows);
        else PyErr_Format(g_error, "%s: %s must be a contiguous %s tensor of shape (%lld, %lld)", what, name, type_name(dtype), (long long) rows, (long long) cols);
        return -1;
    }
    return 0;
}

static int is_f32(const char* what, const char* name, const tensor* t)
{
    if (t->dtype == T_FLOAT) return 1;
    if (t->dtype == T_HALF) return 0;
    return fail(what, name, "must be fp16 or fp32");
}

static int same_device(const char* what, const tensor* const* ts, int n)
{
    const int dev = ts[0]->dev;
    for (int i = 1; i < n; ++i)
        if (ts[i]->given && ts[i]->dev != dev) {
            PyErr_Format(g_error, "%s: the tensors are on devices %d and %d", what, dev, ts[i]->dev);
            return -1;
        }
    const int current = berth_device_current();
    if (dev != current) {
        PyErr_Format(g_error, "%s: the tensors are on device %d, the current device is %d", what, dev, current);
        return -1;
    }
    return 0;
}

/* numbers: errors stay with PyErr_Occurred */
static int to_int(PyObject* o, const char* what, const char* name)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) return -1;
    if (v < INT32_MIN || v > INT32_MAX) return fail(what, name, "is out of range");
    return (int) v;
}
static void* to_stream(PyObject* o) { return o == Py_None ? NULL : PyLong_AsVoidPtr(o); }

/* The library's call without the interpreter's lock: a launch waits where the device's queue is full or its code is still to be loaded,
 * and what the stream waits for may be a peer whose thread needs the lock. */
#define UNLOCKED(rc, call)         \
    do {                           \
        Py_BEGIN_ALLOW_THREADS     \
        rc = (call);               \
        Py_END_ALLOW_THREADS       \
    } while (0)

static PyObject* answer(int rc, const char* what, const char* (*last)(void))
{
    if (rc == 0) Py_RETURN_NONE;
    const char* msg = last();
    if (msg && *msg) PyErr_SetString(g_error, msg);
    else PyErr_Format(g_error, "%s launch failed (%d)", what, rc);
    return NULL;
}

static int arity(const char* what, Py_ssize_t n, Py_ssize_t want)
{
    if (n == want && g_error) return 0;
    PyErr_Format(PyExc_TypeError, "_bind.%s takes %zd arguments, got %zd", what, want, n);
    return -1;
}

/* q or k with its output and norm */
static int read_rows(PyObject* x, PyObject* y, PyObject* norm, const char* name, const char* out_name, const char* norm_name, tensor t[3], berth_rope_rows* rows)
{
    if (read_tensor(x, "rope", name, 3, 0, &t[0]) || read_tensor(y, "rope", out_name, 3, 0, &t[1])) return -1;
    if (t[1].dtype != t[0].dtype || t[1].shape[0] != t[0].shape[0] || t[1].shape[1] != t[0].shape[1] || t[1].shape[2] != t[0].shape[2])
        return fail("rope", out_name, "must have the type and shape of its input");
    if (read_flat(norm, "rope", norm_name, T_BFLOAT16, 1, t[0].shape[2], 0, &t[2])) return -1;
    if (t[0].shape[0] > INT32_MAX || t[0].shape[1] > INT32_MAX || t[0].shape[2] > INT32_MAX) return fail("rope", name, "is too large");
    rows->x = t[0].ptr;
    rows->y = t[1].ptr;
    rows->norm = t[2].given ? t[2].ptr : NULL;
    rows->x_token = t[0].stride[0];
    rows->x_head = t[0].stride[1];
    rows->y_token = t[1].stride[0];
    rows->y_head = t[1].stride[1];
    rows->heads = (int) t[0].shape[1];
    return 0;
}

/* rope(q, k, positions, inv_freq, q_out, k_out, interleaved, attention_factor, q_norm, k_norm, norm_epsilon, norm_bias, stream) */
static PyObject* py_rope(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    (void) self;
    if (arity("rope", n, 13)) return NULL;
    tensor q[3], k[3], pos, freq;
    berth_rope_rows rq, rk;
    if (read_rows(a[0], a[4], a[8], "q", "q_out", "q_norm", q, &rq)) return NULL;
    const int f32 = is_f32("rope", "q", &q[0]);
    if (f32 < 0) return NULL;
    const int has_k = a[1] != Py_None;
    if (has_k) {
        if (read_rows(a[1], a[5], a[9], "k", "k_out", "k_norm", k, &rk)) return NULL;
        if (k[0].dtype != q[0].dtype || k[0].shape[0] != q[0].shape[0] || k[0].shape[2] != q[0].shape[2]) {
            fail("rope", "k", "must share type, tokens and head_dim with q");
            return NULL;
        }
    } else if (a[5] != Py_None || a[9] != Py_None) {
        fail("rope", "k, k_out and k_norm", "go together");
        return NULL;
    }
    if (read_tensor(a[2], "rope", "positions", 1, 0, &pos) || read_tensor(a[3], "rope", "inv_freq", 1, 0, &freq)) return NULL;
    if (pos.dtype != T_INT32 || pos.shape[0] != q[0].shape[0]) {
        fail("rope", "positions", "must be a contiguous int32 tensor with one entry per token");
        return NULL;
    }
    if (freq.dtype != T_DOUBLE || freq.shape[0] > 256) {
        fail("rope", "inv_freq", "must be a contiguous float64 tensor of at most 256 entries");
        return NULL;
    }
    const tensor* ts[8] = {&q[0], &q[1], &q[2], &pos, &freq, &k[0], &k[1], &k[2]};
    if (same_device("rope", ts, has_k ? 8 : 5)) return NULL;
    const int interleaved = PyObject_IsTrue(a[6]);
    const double factor = PyFloat_AsDouble(a[7]), eps = PyFloat_AsDouble(a[10]), bias = PyFloat_AsDouble(a[11]);
    void* stream = to_stream(a[12]);
    if (interleaved < 0 || PyErr_Occurred()) return NULL;
    int rc;
    UNLOCKED(rc, berth_ops_rope(&rq, has_k ? &rk : NULL, pos.ptr, freq.ptr, (int) q[0].shape[0], (int) q[0].shape[2], 2 * (int) freq.shape[0], interleaved,
                                (float) factor, (float) eps, (float) bias, f32, stream));
    return answer(rc, "rope", berth_ops_last_error);
}

/* logprobs(logits, tokens, logprob, rank, entropy, top_idx, top_logprob, vocab or None, inv_temp, stream) */
static PyObject* py_logprobs(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    (void) self;
    const char* what = "logprobs";
    if (arity(what, n, 10)) return NULL;
    tensor x, token, lp, rank, entropy, top, top_lp;
    if (read_tensor(a[0], what, "logits", 2, 0, &x)) return NULL;
    const int f32 = is_f32(what, "logits", &x);
    if (f32 < 0) return NULL;
    const int64_t rows = x.shape[0];
    if (rows > INT32_MAX || x.shape[1] > INT32_MAX) {
        fail(what, "logits", "is too large");
        return NULL;
    }
    const int vocab = a[7] == Py_None ? (int) x.shape[1] : to_int(a[7], what, "vocab");
    if (PyErr_Occurred()) return NULL;
    if (vocab > x.shape[1]) {
        PyErr_Format(g_error, "logprobs: vocab %d exceeds the %lld columns of logits", vocab, (long long) x.shape[1]);
        return NULL;
    }
    if (read_flat(a[1], what, "tokens", T_INT32, 1, rows, 0, &token) || read_flat(a[2], what, "logprob", T_FLOAT, 1, rows, 0, &lp) ||
        read_flat(a[3], what, "rank", T_INT32, 1, rows, 0, &rank) || read_flat(a[4], what, "entropy", T_FLOAT, 1, rows, 0, &entropy))
        return NULL;
    int64_t best = 0;
    if ((a[5] == Py_None) != (a[6] == Py_None)) {
        fail(what, "top_idx and top_logprob", "go together");
        return NULL;
    }
    top.given = top_lp.given = 0;
    if (a[5] != Py_None) {
        if (read_tensor(a[5], what, "top_idx", 2, 0, &top)) return NULL;
        best = top.shape[1];
        if (best > INT32_MAX) {
            fail(what, "top_idx", "is too large");
            return NULL;
        }
        if (read_flat(a[5], what, "top_idx", T_INT32, 2, rows, best, &top) || read_flat(a[6], what, "top_logprob", T_FLOAT, 2, rows, best, &top_lp)) return NULL;
    }
    const tensor* ts[7] = {&x, &token, &lp, &rank, &entropy, &top, &top_lp};
    if (same_device(what, ts, 7)) return NULL;
    const double inv_temp = PyFloat_AsDouble(a[8]);
    void* stream = to_stream(a[9]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    UNLOCKED(rc, berth_ops_logprobs(x.ptr, f32, x.stride[0], token.given ? token.ptr : NULL, (float) inv_temp, lp.given ? lp.ptr : NULL,
                                    rank.given ? rank.ptr : NULL, entropy.given ? entropy.ptr : NULL, best ? top.ptr : NULL, best ? top_lp.ptr : NULL,
                                    (int) best, (int) rows, vocab, stream));
    return answer(rc, what, berth_ops_last_error);
}

/* route(logits, selection_bias, topk_idx, topk_w, top_k, score, n_group, topk_group, group_score, renormalize, scale, stream) */
static PyObject* py_route(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    (void) self;
    const char* what = "moe route";
    if (arity("route", n, 12)) return NULL;
    tensor x, bias, idx, w;
    if (read_tensor(a[0], what, "logits", 2, 0, &x)) return NULL;
    const int f32 = is_f32(what, "logits", &x);
    if (f32 < 0) return NULL;
    const int64_t rows = x.shape[0], experts = x.shape[1];
    if (rows > INT32_MAX || experts > INT32_MAX) {
        fail(what, "logits", "is too large");
        return NULL;
    }
    const int k = to_int(a[4], what, "top_k"), score = to_int(a[5], what, "score"), groups = to_int(a[6], what, "n_group"), kept = to_int(a[7], what, "topk_group"),
              group_score = to_int(a[8], what, "group_score"), renormalize = PyObject_IsTrue(a[9]);
    const double scale = PyFloat_AsDouble(a[10]);
    void* stream = to_stream(a[11]);
    if (PyErr_Occurred()) return NULL;
    if (read_flat(a[1], what, "selection_bias", T_FLOAT, 1, experts, 0, &bias) || read_flat(a[2], what, "topk_idx", T_INT32, 2, rows, k, &idx) ||
        read_flat(a[3], what, "topk_w", T_FLOAT, 2, rows, k, &w))
        return NULL;
    const tensor* ts[4] = {&x, &bias, &idx, &w};
    if (same_device(what, ts, 4)) return NULL;
    int rc;
    UNLOCKED(rc, berth_moe_route(x.ptr, f32, x.stride[0], bias.given ? bias.ptr : NULL, idx.given ? idx.ptr : NULL, w.given ? w.ptr : NULL, (int) rows,
                                 (int) experts, k, score, groups, kept, group_score, renormalize, (float) scale, stream));
    return answer(rc, what, berth_moe_last_error);
}

#define NEEDS "rope, logprobs and route read tensors through: torch 2.11 publishes it"
/* init(Error, torch.Tensor): the exception to raise and the class of the tensors */
static PyObject* py_init(PyObject* self, PyObject* const* a, Py_ssize_t n)
{
    (void) self;
    if (n != 2 || !PyType_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "_bind.init takes (Error, torch.Tensor)");
        return NULL;
    }
    PyObject* capsule = PyObject_GetAttrString(a[1], "__dlpack_c_exchange_api__");
    if (!capsule) {
        if (PyErr_ExceptionMatches(PyExc_AttributeError)) {
            PyErr_Clear();
            PyErr_Format(PyExc_ImportError, "%s has no __dlpack_c_exchange_api__ (DLPack 1.x), which " NEEDS, ((PyTypeObject*) a[1])->tp_name);
        }
        return NULL;
    }
    const dl_exchange* x = (const dl_exchange*) PyCapsule_GetPointer(capsule, "dlpack_exchange_api");   /* lives as long as torch */
    Py_DECREF(capsule);
    if (!x) return NULL;
    if (x->version.major != 1 || !x->tensor_from_object) {
        PyErr_Format(PyExc_ImportError, "%s offers an exchange interface of DLPack %d.%d; version 1.x " NEEDS, ((PyTypeObject*) a[1])->tp_name,
                     (int) x->version.major, (int) x->version.minor);
        return NULL;
    }
    g_exchange = x;
    Py_XSETREF(g_tensor, (PyTypeObject*) Py_NewRef(a[1]));
    Py_XSETREF(g_error, Py_NewRef(a[0]));
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"init", (PyCFunction) (void (*)(void)) py_init, METH_FASTCALL, NULL},
                                {"rope", (PyCFunction) (void (*)(void)) py_rope, METH_FASTCALL, NULL},
                                {"logprobs", (PyCFunction) (void (*)(void)) py_logprobs, METH_FASTCALL, NULL},
                                {"route", (PyCFunction) (void (*)(void)) py_route, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Callers of rope, logprobs and route over torch tensors.", -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__bind(void)
{
    return PyModule_Create(&module);
}
