/* CPython side of the serving operators (chatterbox_amd/ops.py): torch tensors to the structs of include/t3mi.h.
 *
 * A decode step calls these operators on a few rows, where the GPU needs 3-10 us and taking tensors apart in Python code took 12-17: the
 * attributes are read here instead: by torch's DLPack exchange table where it has one (a tensor in 0.05 us), by the tensors' methods
 * otherwise (0.4 us); nothing of torch is linked.  What a tensor has to be is checked here, with ValueError; what the sizes have to be is
 * checked by the C entry points, whose status goes to _lib.check.
 * The entry points' addresses come from the ctypes binding (bind), so that this module and it use one library. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "t3mi.h"

#ifdef T3MI_DLPACK
#include <ATen/dlpack.h>
static int (*f_dltensor)(void*, DLTensor*);   /* of torch's table, or NULL */
static PyObject* t_tensor;
#endif

static int (*f_append)(const t3mi_paged_cache*, const t3mi_append_args*, void*);
static int (*f_workspace)(const t3mi_paged_cache*, const t3mi_attention_args*, size_t*);
static int (*f_attention)(const t3mi_paged_cache*, const t3mi_attention_args*, void*);
static int (*f_logits)(const t3mi_logits_args*, void*);

/* of torch, and _lib.check */
static PyObject *t_f32, *t_bf16, *t_i32, *c_empty, *c_empty_like, *c_stream, *c_grad, *c_check, *c_forward, *c_unpack;
static PyObject *s_data_ptr, *s_dtype, *s_get_device, *s_shape, *s_stride, *s_requires_grad, *s_device, *s_new_empty, *s_level, *s_tangent, *kw_dtype_device;

enum { F32 = 1, BF16 = 2, I32 = 4 };
#define MAXD 4
typedef struct {
    void* p;
    int dtype, device, dim;
    int64_t shape[MAXD], stride[MAXD];
} Ten;

static int code_of(const Ten* t) { return t->dtype == BF16 ? T3MI_W_BF16 : T3MI_W_F32; }

static int ints_of(PyObject* tuple, int64_t* o, int dim) {
    for (int i = 0; i < dim; ++i) {
        o[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
        if (o[i] == -1 && PyErr_Occurred()) return -1;
    }
    return 0;
}

static const char* word_of(int types) { return types == I32 ? "int32" : types == F32 ? "float32" : "float32 or bfloat16"; }

static int need_gpu(const char* name, int device, int wanted_device) {
    if (device < 0)
        PyErr_Format(PyExc_ValueError, "%s is on the host: the operators run on the GPU, and all tensors of a call are on the same one", name);
    else if (wanted_device >= 0 && device != wanted_device)
        PyErr_Format(PyExc_ValueError, "%s is on GPU %d, not on GPU %d", name, device, wanted_device);
    else
        return 0;
    return -1;
}

/* forward mode: whether a level is open (asked once a call), and whether t carries a tangent of it */
static int level_open;
static int look_for_level(void) {
    PyObject* r = PyObject_GetAttr(c_forward, s_level);
    if (!r) return -1;
    const long level = PyLong_AsLong(r);
    Py_DECREF(r);
    if (level == -1 && PyErr_Occurred()) return -1;
    level_open = level >= 0;
    return 0;
}
static int wants_no_tangent(const char* name, PyObject* t) {
    if (!level_open) return 0;
    PyObject* r = PyObject_CallOneArg(c_unpack, t);
    PyObject* d = r ? PyObject_GetAttr(r, s_tangent) : NULL;
    Py_XDECREF(r);
    if (!d) return -1;
    const int none = d == Py_None;
    Py_DECREF(d);
    if (!none) PyErr_Format(PyExc_ValueError, "%s carries a forward-mode gradient: this operator has none", name);
    return none ? 0 : -1;
}

static int wants_no_gradient(const char* name, PyObject* t) {
    PyObject* r = PyObject_GetAttr(t, s_requires_grad);
    if (!r) return -1;
    const int grad = PyObject_IsTrue(r);
    Py_DECREF(r);
    if (grad < 0) return grad;
    if (!grad) return wants_no_tangent(name, t);
    if (!(r = PyObject_CallNoArgs(c_grad))) return -1;
    const int on = PyObject_IsTrue(r);
    Py_DECREF(r);
    if (on > 0) PyErr_Format(PyExc_ValueError, "%s requires gradients: this operator has no backward pass", name);
    return on ? -1 : wants_no_tangent(name, t);
}

#ifdef T3MI_DLPACK
/* `take` by the exchange table: 1 if it could say nothing about this object (the methods then do) */
static int take_dl(const char* name, PyObject* t, int types, int dim, int device, Ten* o) {
    DLTensor d;
    if (!f_dltensor || !PyObject_TypeCheck(t, (PyTypeObject*)t_tensor)) return 1;
    if (f_dltensor(t, &d)) {
        PyErr_Clear();
        return 1;
    }
    o->device = d.device.device_type == kDLROCM || d.device.device_type == kDLCUDA ? d.device.device_id : -1;
    if (need_gpu(name, o->device, device)) return -1;
    const DLDataType y = d.dtype;
    o->dtype = y.lanes != 1 ? 0 : y.code == kDLFloat && y.bits == 32 ? F32 : y.code == kDLBfloat && y.bits == 16 ? BF16 : y.code == kDLInt && y.bits == 32 ? I32 : 0;
    if (!(o->dtype & types) || d.ndim != dim || !d.strides) return 1;   /* (the methods find the words) */
    for (int i = 0; i < dim; ++i) {
        o->shape[i] = d.shape[i];
        o->stride[i] = d.strides[i];
    }
    o->dim = dim;
    o->p = d.data ? (char*)d.data + d.byte_offset : NULL;
    return 0;
}
#endif

static int take_methods(const char* name, PyObject* t, int types, int dim, int device, Ten* o);

/* A tensor of `dim` dimensions on GPU `device` (-1: any GPU) of one of `types`, its last dimension contiguous, no gradients asked for.
 * A dimension of one entry has no stride worth the name: 0. */
static int take(const char* name, PyObject* t, int types, int dim, int device, Ten* o) {
    int rc = 1;
#ifdef T3MI_DLPACK
    rc = take_dl(name, t, types, dim, device, o);
#endif
    if (rc > 0) rc = take_methods(name, t, types, dim, device, o);
    if (rc) return -1;
    if (o->stride[dim - 1] != 1 && o->shape[dim - 1] > 1) {
        PyErr_Format(PyExc_ValueError, "%s: the last dimension must be contiguous", name);
        return -1;
    }
    for (int i = 0; i < dim; ++i)
        if (o->shape[i] <= 1) o->stride[i] = 0;
    return types == I32 ? 0 : wants_no_gradient(name, t);
}

static int take_methods(const char* name, PyObject* t, int types, int dim, int device, Ten* o) {
    PyObject* r = PyObject_CallMethodNoArgs(t, s_get_device);
    if (!r) return -1;
    o->device = (int)PyLong_AsLong(r);
    Py_DECREF(r);
    if (o->device == -1 && PyErr_Occurred()) return -1;
    if (need_gpu(name, o->device, device)) return -1;
    if (!(r = PyObject_GetAttr(t, s_dtype))) return -1;
    o->dtype = r == t_f32 ? F32 : r == t_bf16 ? BF16 : r == t_i32 ? I32 : 0;
    if (!(o->dtype & types)) PyErr_Format(PyExc_ValueError, "%s has dtype %S: %s wanted", name, r, word_of(types));
    Py_DECREF(r);
    if (!(o->dtype & types)) return -1;
    if (!(r = PyObject_GetAttr(t, s_shape))) return -1;
    if (!PyTuple_Check(r) || PyTuple_GET_SIZE(r) != dim) {
        PyErr_Format(PyExc_ValueError, "%s must have %d dimensions, its shape is %R", name, dim, r);
        Py_DECREF(r);
        return -1;
    }
    o->dim = dim;
    int bad = ints_of(r, o->shape, dim);
    Py_DECREF(r);
    if (bad || !(r = PyObject_CallMethodNoArgs(t, s_stride))) return -1;
    bad = !PyTuple_Check(r) || PyTuple_GET_SIZE(r) != dim || ints_of(r, o->stride, dim);
    Py_DECREF(r);
    if (bad) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s has no strides", name);
        return -1;
    }
    if (!(r = PyObject_CallMethodNoArgs(t, s_data_ptr))) return -1;
    o->p = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return PyErr_Occurred() ? -1 : 0;
}

static int says(PyObject* exc, const char* fmt, const char* name, long long a, long long b) {
    PyErr_Format(exc, fmt, name, a, b);
    return -1;
}

/* an int32 [n] or None */
static int take_list(const char* name, PyObject* t, int64_t n, int device, const int32_t** o) {
    Ten x;
    *o = NULL;
    if (t == Py_None) return 0;
    if (take(name, t, I32, 1, device, &x)) return -1;
    if (x.shape[0] != n) return says(PyExc_ValueError, "%s has shape (%lld,), wanted (%lld,)", name, x.shape[0], n);
    *o = x.p;
    return 0;
}

static int take_cache(PyObject* k, PyObject* v, PyObject* table, t3mi_paged_cache* c, Ten* kt) {
    Ten vt, tt;
    if (take("k_pages", k, F32 | BF16, 4, -1, kt) || take("v_pages", v, F32 | BF16, 4, kt->device, &vt) || take("block_table", table, I32, 2, kt->device, &tt)) return -1;
    if (vt.dtype != kt->dtype) {
        PyErr_SetString(PyExc_ValueError, "v_pages and k_pages differ in dtype");
        return -1;
    }
    for (int i = 0; i < 4; ++i)
        if (vt.shape[i] != kt->shape[i]) return says(PyExc_ValueError, "%s: k_pages and v_pages differ in shape (%lld, %lld)", "v_pages", kt->shape[i], vt.shape[i]);
    for (int i = 0; i < 4; ++i)
        if (kt->shape[i] > INT32_MAX) return says(PyExc_ValueError, "%s: an extent of %lld is more than %lld", "k_pages", kt->shape[i], INT32_MAX);
    if (tt.shape[0] > INT32_MAX || tt.shape[1] > INT32_MAX) return says(PyExc_ValueError, "%s: %lld x %lld entries", "block_table", tt.shape[0], tt.shape[1]);
    c->k = kt->p;
    c->v = vt.p;
    for (int i = 0; i < 3; ++i) { c->k_stride[i] = kt->stride[i]; c->v_stride[i] = vt.stride[i]; }
    c->block_table = tt.p;
    c->table_stride = tt.stride[0];
    c->n_seqs = (int32_t)tt.shape[0];
    c->max_pages = (int32_t)tt.shape[1];
    c->n_pages = (int32_t)kt->shape[0];
    c->page_size = (int32_t)kt->shape[1];
    c->kv_heads = (int32_t)kt->shape[2];
    c->head_dim = (int32_t)kt->shape[3];
    c->dtype = code_of(kt);
    c->device = kt->device;
    return 0;
}

/* a new tensor like `like` (contiguous), or of another type */
static PyObject* fresh(PyObject* like, const Ten* t, PyObject* dtype, int same) {
    int64_t run = 1;
    int dense = 1;
    for (int i = t->dim - 1; i >= 0; --i) {
        if (t->shape[i] > 1 && t->stride[i] != run) dense = 0;
        run *= t->shape[i];
    }
    if (same && dense) return PyObject_CallOneArg(c_empty_like, like);
    PyObject* shape = PyObject_GetAttr(like, s_shape);
    PyObject* dev = shape ? PyObject_GetAttr(like, s_device) : NULL;
    PyObject* r = NULL;
    if (dev) {
        PyObject* args[3] = {shape, dtype, dev};
        r = PyObject_Vectorcall(c_empty, args, 1, kw_dtype_device);
    }
    Py_XDECREF(shape);
    Py_XDECREF(dev);
    return r;
}

static int stream_of(int device, void** s) {
    PyObject* d = PyLong_FromLong(device);
    PyObject* r = d ? PyObject_CallOneArg(c_stream, d) : NULL;
    Py_XDECREF(d);
    if (!r) return -1;
    *s = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return PyErr_Occurred() ? -1 : 0;
}

/* `out` (owned) after a call that returned rc: itself, or the error that _lib.check raises */
static PyObject* result(int rc, PyObject* out) {
    if (rc) {
        PyObject* r = PyObject_CallFunction(c_check, "i", rc);
        if (!r) {
            Py_XDECREF(out);
            return NULL;
        }
        Py_DECREF(r);
    }
    if (out) return out;
    Py_RETURN_NONE;
}

static int wanted(const char* f, Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return 0;
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", f, want, n);
    return -1;
}

/* append(k, v, k_pages, v_pages, block_table, positions, seq, q, q_out, cos, sin) -> q_out */
static PyObject* py_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    t3mi_paged_cache c;
    t3mi_append_args g = {0};
    Ten kc, k, v, q, o, cs, sn;
    if (wanted("append", n, 11) || look_for_level() || take_cache(a[2], a[3], a[4], &c, &kc)) return NULL;
    if (take("k", a[0], F32 | BF16, 3, kc.device, &k) || take("v", a[1], k.dtype, 3, kc.device, &v)) return NULL;
    const int64_t rows = k.shape[0];
    if (rows > INT32_MAX || v.shape[0] != rows || k.shape[1] != c.kv_heads || v.shape[1] != c.kv_heads || k.shape[2] != c.head_dim || v.shape[2] != c.head_dim) {
        PyErr_Format(PyExc_ValueError, "k and v must have shape [rows, %d, %d]", c.kv_heads, c.head_dim);
        return NULL;
    }
    if (a[5] == Py_None) {
        PyErr_SetString(PyExc_ValueError, "positions is None");
        return NULL;
    }
    if (take_list("positions", a[5], rows, kc.device, &g.positions) || take_list("seq", a[6], rows, kc.device, &g.seq)) return NULL;
    g.k = k.p; g.v = v.p;
    g.k_stride[0] = k.stride[0]; g.k_stride[1] = k.stride[1]; g.v_stride[0] = v.stride[0]; g.v_stride[1] = v.stride[1];
    g.rows = (int32_t)rows;
    g.dtype = code_of(&k);
    if (a[9] != Py_None || a[10] != Py_None) {
        if (take("cos", a[9], F32, 2, kc.device, &cs) || take("sin", a[10], F32, 2, kc.device, &sn)) return NULL;
        if (cs.shape[0] != sn.shape[0] || cs.shape[1] != sn.shape[1] || cs.stride[0] != sn.stride[0] || cs.shape[1] < c.head_dim / 2 || cs.shape[0] > INT32_MAX) {
            PyErr_Format(PyExc_ValueError, "cos and sin must be alike, [positions, >= %d]", c.head_dim / 2);
            return NULL;
        }
        g.cos = cs.p; g.sin = sn.p; g.rope_stride = cs.stride[0]; g.rope_len = (int32_t)cs.shape[0];
    }
    PyObject* out = NULL;
    if (a[7] != Py_None) {
        if (take("q", a[7], k.dtype, 3, kc.device, &q)) return NULL;
        if (q.shape[0] != rows || q.shape[2] != c.head_dim || q.shape[1] > INT32_MAX) {
            PyErr_Format(PyExc_ValueError, "q must have shape [%lld, heads, %d]", (long long)rows, c.head_dim);
            return NULL;
        }
        if (a[8] == Py_None) out = fresh(a[7], &q, k.dtype == BF16 ? t_bf16 : t_f32, 1);
        else Py_INCREF(out = a[8]);
        if (!out || take("q_out", out, k.dtype, 3, kc.device, &o)) goto fail;
        if (o.shape[0] != rows || o.shape[1] != q.shape[1] || o.shape[2] != c.head_dim) {
            PyErr_SetString(PyExc_ValueError, "q_out must have the shape of q");
            goto fail;
        }
        g.q = q.p; g.q_out = o.p; g.q_heads = (int32_t)q.shape[1];
        g.q_stride[0] = q.stride[0]; g.q_stride[1] = q.stride[1]; g.q_out_stride[0] = o.stride[0]; g.q_out_stride[1] = o.stride[1];
        if (!g.q && rows == 0) g.q_out = NULL;
    } else if (a[8] != Py_None) {
        PyErr_SetString(PyExc_ValueError, "q_out without q");
        return NULL;
    }
    void* s;
    if (stream_of(kc.device, &s)) goto fail;
    int rc = 0;
    if (rows) {
        Py_BEGIN_ALLOW_THREADS
        rc = f_append(&c, &g, s);
        Py_END_ALLOW_THREADS
    }
    return result(rc, out);
fail:
    Py_XDECREF(out);
    return NULL;
}

/* attention(q, k_pages, v_pages, block_table, lengths, seq, starts, scale or None, max_length, out, out_dtype, prompt: 1, 0 or -1) -> out */
static PyObject* py_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    t3mi_paged_cache c;
    t3mi_attention_args g = {0};
    Ten kc, q, o;
    if (wanted("attention", n, 12) || look_for_level() || take_cache(a[1], a[2], a[3], &c, &kc) || take("q", a[0], F32 | BF16, 3, kc.device, &q)) return NULL;
    const int64_t rows = q.shape[0];
    if (rows > INT32_MAX || q.shape[1] > INT32_MAX || q.shape[2] != c.head_dim) {
        PyErr_Format(PyExc_ValueError, "q has head_dim %lld, the cache %d", (long long)q.shape[2], c.head_dim);
        return NULL;
    }
    if (a[4] == Py_None) {
        PyErr_SetString(PyExc_ValueError, "lengths is None");
        return NULL;
    }
    if (take_list("lengths", a[4], rows, kc.device, &g.lengths) || take_list("seq", a[5], rows, kc.device, &g.seq) ||
        take_list("starts", a[6], rows, kc.device, &g.starts))
        return NULL;
    g.scale = c.head_dim == 64 ? 0.125f : 0.08838834764831845f;
    if (a[7] != Py_None) {
        g.scale = (float)PyFloat_AsDouble(a[7]);
        if (PyErr_Occurred()) return NULL;
    }
    const long most = PyLong_AsLong(a[8]);
    if (most == -1 && PyErr_Occurred()) return NULL;
    g.max_length = most > INT32_MAX ? INT32_MAX : most < 0 ? -1 : (int32_t)most;
    g.prompt = (int32_t)PyLong_AsLong(a[11]);
    if (PyErr_Occurred()) return NULL;
    PyObject *out = NULL, *ws = NULL;
    if (a[9] == Py_None) {
        if (a[10] != Py_None && a[10] != t_f32 && a[10] != t_bf16) {
            PyErr_Format(PyExc_ValueError, "out_dtype is %S: float32 or bfloat16 wanted", a[10]);
            return NULL;
        }
        PyObject* own = q.dtype == BF16 ? t_bf16 : t_f32;
        out = fresh(a[0], &q, a[10] == Py_None ? own : a[10], a[10] == Py_None || a[10] == own);
    } else {
        Py_INCREF(out = a[9]);
    }
    if (!out || take("out", out, F32 | BF16, 3, kc.device, &o)) goto fail;
    if (o.shape[0] != rows || o.shape[1] != q.shape[1] || o.shape[2] != q.shape[2] || (a[10] != Py_None && a[10] != (o.dtype == BF16 ? t_bf16 : t_f32))) {
        PyErr_SetString(PyExc_ValueError, "out must have the shape of q, and out_dtype where that is given");
        goto fail;
    }
    g.q = q.p; g.out = o.p;
    g.q_stride[0] = q.stride[0]; g.q_stride[1] = q.stride[1]; g.out_stride[0] = o.stride[0]; g.out_stride[1] = o.stride[1];
    g.rows = (int32_t)rows;
    g.q_heads = (int32_t)q.shape[1];
    g.q_dtype = code_of(&q);
    g.out_dtype = code_of(&o);
    int rc = f_workspace(&c, &g, &g.workspace_bytes);
    if (rc || rows == 0) return result(rc, out);
    if (g.workspace_bytes) {
        /* (of q's type and on its device: the cheapest way to ask torch for memory) */
        PyObject* size = PyLong_FromSize_t((g.workspace_bytes + 3) / (q.dtype == BF16 ? 2 : 4));
        ws = size ? PyObject_CallMethodOneArg(a[0], s_new_empty, size) : NULL;
        Py_XDECREF(size);
        PyObject* r = ws ? PyObject_CallMethodNoArgs(ws, s_data_ptr) : NULL;
        if (!r) goto fail;
        g.workspace = PyLong_AsVoidPtr(r);
        Py_DECREF(r);
        if (PyErr_Occurred()) goto fail;
    }
    void* s;
    if (stream_of(kc.device, &s)) goto fail;
    Py_BEGIN_ALLOW_THREADS
    rc = f_attention(&c, &g, s);
    Py_END_ALLOW_THREADS
    Py_XDECREF(ws);   /* (torch's allocator gives its memory to later work of the same stream alone) */
    return result(rc, out);
fail:
    Py_XDECREF(ws);
    Py_XDECREF(out);
    return NULL;
}

/* a penalty: a number, or float32 [rows] */
static int take_each(const char* name, PyObject* x, int64_t rows, int device, float* number, const float** each) {
    Ten t;
    *each = NULL;
    *number = 1.f;
    if (PyFloat_Check(x) || PyLong_Check(x) || !PyObject_HasAttr(x, s_get_device)) {   /* (numbers of other libraries, too) */
        *number = (float)PyFloat_AsDouble(x);
        return PyErr_Occurred() ? -1 : 0;
    }
    if (take(name, x, F32, 1, device, &t)) return -1;
    if (t.shape[0] != rows) return says(PyExc_ValueError, "%s has %lld entries for %lld rows", name, t.shape[0], rows);
    *each = t.p;
    return 0;
}

/* logits(logits, uncond, cfg_weight, tokens, n_tokens, repetition, frequency, presence, bias_ids, bias_values, allowed, out) -> out */
static PyObject* py_logits(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    t3mi_logits_args g = {0};
    Ten l, u, t, x, y, o;
    if (wanted("logits", n, 12) || look_for_level() || take("logits", a[0], F32 | BF16, 2, -1, &l)) return NULL;
    const int64_t rows = l.shape[0], vocab = l.shape[1];
    if (rows > INT32_MAX || vocab > INT32_MAX) {
        PyErr_SetString(PyExc_ValueError, "logits has too many rows or entries");
        return NULL;
    }
    g.cfg_weight = (float)PyFloat_AsDouble(a[2]);
    if (PyErr_Occurred()) return NULL;
    if (a[1] != Py_None) {
        if (take("uncond", a[1], l.dtype, 2, l.device, &u)) return NULL;
        if (u.shape[0] != rows || u.shape[1] != vocab) {
            PyErr_SetString(PyExc_ValueError, "uncond must have the shape of logits");
            return NULL;
        }
        g.uncond = u.p; g.uncond_stride = u.stride[0];
    }
    if ((a[3] == Py_None) != (a[4] == Py_None) || (a[8] == Py_None) != (a[9] == Py_None)) {
        PyErr_SetString(PyExc_ValueError, "tokens and n_tokens go together, and bias_ids and bias_values");
        return NULL;
    }
    if (a[3] != Py_None) {
        if (take("tokens", a[3], I32, 2, l.device, &t) || take_list("n_tokens", a[4], rows, l.device, &g.n_tokens)) return NULL;
        if (t.shape[0] != rows || t.shape[1] > INT32_MAX) {
            says(PyExc_ValueError, "%s has %lld rows, wanted %lld", "tokens", t.shape[0], rows);
            return NULL;
        }
        g.tokens = t.p; g.tokens_stride = t.stride[0]; g.token_cap = (int32_t)t.shape[1];
        if (!g.token_cap) g.tokens = NULL;
    }
    if (take_each("repetition_penalty", a[5], rows, l.device, &g.repetition, &g.repetition_each) ||
        take_each("frequency_penalty", a[6], rows, l.device, &g.frequency, &g.frequency_each) ||
        take_each("presence_penalty", a[7], rows, l.device, &g.presence, &g.presence_each))
        return NULL;
    if (a[8] != Py_None) {
        if (take("bias_ids", a[8], I32, 2, l.device, &x) || take("bias_values", a[9], F32, 2, l.device, &y)) return NULL;
        if (x.shape[0] != y.shape[0] || x.shape[1] != y.shape[1] || (x.shape[0] != 1 && x.shape[0] != rows) || x.shape[1] > INT32_MAX) {
            PyErr_Format(PyExc_ValueError, "bias_ids and bias_values must have shape [%lld or 1, n]", (long long)rows);
            return NULL;
        }
        g.bias_ids = x.p; g.bias_values = y.p; g.n_bias = (int32_t)x.shape[1];
        g.bias_ids_stride = x.stride[0]; g.bias_values_stride = y.stride[0];   /* (0 for a single row) */
    }
    if (a[10] != Py_None) {
        if (take("allowed", a[10], I32, 2, l.device, &x)) return NULL;
        if ((x.shape[0] != 1 && x.shape[0] != rows) || x.shape[1] < (vocab + 31) / 32) {
            PyErr_Format(PyExc_ValueError, "allowed must have shape [%lld or 1, >= %lld]", (long long)rows, (long long)(vocab + 31) / 32);
            return NULL;
        }
        g.allowed = x.p; g.allowed_stride = x.stride[0];
    }
    PyObject* out = NULL;
    if (a[11] == Py_None) out = fresh(a[0], &l, l.dtype == BF16 ? t_bf16 : t_f32, 1);
    else Py_INCREF(out = a[11]);
    if (!out || take("out", out, l.dtype, 2, l.device, &o)) goto fail;
    if (o.shape[0] != rows || o.shape[1] != vocab) {
        PyErr_SetString(PyExc_ValueError, "out must have the shape of logits");
        goto fail;
    }
    g.logits = l.p; g.logits_stride = l.stride[0];
    g.out = o.p; g.out_stride = o.stride[0];
    g.rows = (int32_t)rows; g.vocab = (int32_t)vocab; g.dtype = code_of(&l); g.device = l.device;
    void* s;
    if (stream_of(l.device, &s)) goto fail;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f_logits(&g, s);
    Py_END_ALLOW_THREADS
    return result(rc, out);
fail:
    Py_XDECREF(out);
    return NULL;
}

/* bind(4 addresses, float32, bfloat16, int32, empty, empty_like, raw stream of a device, is_grad_enabled, check, torch.autograd.forward_ad, its
 * unpack_dual, torch.Tensor, its DLPack exchange capsule or None) */
static PyObject* py_bind(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (wanted("bind", n, 16)) return NULL;
    void* p[4];
    for (int i = 0; i < 4; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return NULL;
    }
    f_append = (int (*)(const t3mi_paged_cache*, const t3mi_append_args*, void*))p[0];
    f_workspace = (int (*)(const t3mi_paged_cache*, const t3mi_attention_args*, size_t*))p[1];
    f_attention = (int (*)(const t3mi_paged_cache*, const t3mi_attention_args*, void*))p[2];
    f_logits = (int (*)(const t3mi_logits_args*, void*))p[3];
    PyObject** keep[10] = {&t_f32, &t_bf16, &t_i32, &c_empty, &c_empty_like, &c_stream, &c_grad, &c_check, &c_forward, &c_unpack};
    for (int i = 0; i < 10; ++i) {
        Py_INCREF(a[4 + i]);
        Py_XSETREF(*keep[i], a[4 + i]);
    }
#ifdef T3MI_DLPACK
    f_dltensor = NULL;
    if (PyType_Check(a[14]) && PyCapsule_IsValid(a[15], "dlpack_exchange_api")) {
        const DLPackExchangeAPI* x = PyCapsule_GetPointer(a[15], "dlpack_exchange_api");
        if (x->header.version.major == DLPACK_MAJOR_VERSION) {   /* (the table lives as long as torch does) */
            Py_INCREF(a[14]);
            Py_XSETREF(t_tensor, a[14]);
            f_dltensor = x->dltensor_from_py_object_no_sync;
        }
    }
#endif
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))py_bind, METH_FASTCALL, "addresses and torch's objects, once"},
    {"append", (PyCFunction)(void (*)(void))py_append, METH_FASTCALL, "t3mi_paged_append on tensors"},
    {"attention", (PyCFunction)(void (*)(void))py_attention, METH_FASTCALL, "t3mi_paged_attention on tensors"},
    {"logits", (PyCFunction)(void (*)(void))py_logits, METH_FASTCALL, "t3mi_process_logits on tensors"},
    {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", "tensors to the structs of t3mi.h", -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__ops(void) {
    struct { PyObject** o; const char* s; } names[] = {{&s_data_ptr, "data_ptr"}, {&s_dtype, "dtype"}, {&s_get_device, "get_device"}, {&s_shape, "shape"},
                                                        {&s_stride, "stride"}, {&s_requires_grad, "requires_grad"}, {&s_device, "device"}, {&s_new_empty, "new_empty"},
                                                        {&s_level, "_current_level"}, {&s_tangent, "tangent"}};
    for (size_t i = 0; i < sizeof(names) / sizeof(names[0]); ++i)
        if (!(*names[i].o = PyUnicode_InternFromString(names[i].s))) return NULL;
    if (!(kw_dtype_device = Py_BuildValue("(ss)", "dtype", "device"))) return NULL;
    return PyModule_Create(&module);
}
