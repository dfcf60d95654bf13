// The tensor side of the Python binding of the token operators (b2lstm/operators.py): reads addresses, shapes, strides and element types
// from tensor objects, checks them, and calls the library.  A call of an operator on a handful of frames is as long as its host work;
// done attribute by attribute in Python that was half of it.  Knows no tensor library: a tensor is any object with data_ptr(), shape,
// stride(), numel(), is_contiguous(), dtype and is_cuda; one that has get_device() too has to be on the device that the call goes to.  The library's functions come as addresses (bind), so this file links against nothing.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <string.h>

#include "../../include/b2lstm.h"

namespace {

PyObject *g_error = nullptr;      // b2lstm.B2Error
PyObject *g_types = nullptr;      // dtype object -> code
enum { INT32 = 16, BYTE = 17, INT8 = 18, OTHER = 19 };     // BYTE: uint8 and bool, and int8 where bytes are meant

struct Api {
    decltype(&b2_last_error_string) last_error;
    decltype(&b2_current_device) current_device;
    decltype(&b2_embedding_forward) embedding_forward;
    decltype(&b2_embedding_backward) embedding_backward;
    decltype(&b2_block_norm_forward) block_norm_forward;
    decltype(&b2_block_norm_backward) block_norm_backward;
    decltype(&b2_logprob_forward) logprob_forward;
    decltype(&b2_logprob_backward) logprob_backward;
    decltype(&b2_gradient_norm) gradient_norm;
    decltype(&b2_gradient_clip) gradient_clip;
    decltype(&b2_distill_forward) distill_forward;
    decltype(&b2_distill_backward) distill_backward;
    decltype(&b2_beam_select) beam_select;
    decltype(&b2_beam_reorder) beam_reorder;
    decltype(&b2_int8_quantize) int8_quantize;
    decltype(&b2_int8_product) int8_product;
} api;

PyObject *s_shape, *s_stride, *s_dtype, *s_is_cuda, *s_get_device, *s_data_ptr, *s_numel, *s_is_contiguous;

// an owned reference
struct Ref {
    PyObject *p;
    explicit Ref(PyObject *o) : p(o) {}
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
    explicit operator bool() const { return p != nullptr; }
};

bool refuse(const char *fmt, ...) {
    va_list v;
    va_start(v, fmt);
    PyErr_FormatV(g_error ? g_error : PyExc_RuntimeError, fmt, v);
    va_end(v);
    return false;
}

// code of an element type: B2_F32 ..., INT32, BYTE or OTHER; -1 with an exception set
int type_of(const Ref &dtype) {
    if (!dtype) return -1;
    PyObject *known = PyDict_GetItemWithError(g_types, dtype.p);
    if (known) return (int)PyLong_AsLong(known);
    if (PyErr_Occurred()) return -1;
    Ref text(PyObject_Str(dtype.p));
    const char *s = text ? PyUnicode_AsUTF8(text.p) : nullptr;
    if (!s) return -1;
    const char *dot = strrchr(s, '.'), *name = dot ? dot + 1 : s;
    static const struct { const char *name; int code; } known_names[] = {{"float32", B2_F32}, {"bfloat16", B2_BF16}, {"float16", B2_F16}, {"int32", INT32},
                                                                         {"uint8", BYTE}, {"int8", INT8}, {"bool", BYTE}};
    int code = OTHER;
    for (const auto &k : known_names)
        if (!strcmp(name, k.name)) code = k.code;
    Ref value(PyLong_FromLong(code));
    if (!value || PyDict_SetItem(g_types, dtype.p, value.p) < 0) return -1;
    return code;
}

thread_local int t_device;         // of the call under way on this thread
// Kernels run on the current device: memory of another one is out of their reach, or a fault.
bool on_gpu(PyObject *t, const char *name) {
    Ref at(PyObject_CallMethodNoArgs(t, s_get_device));
    if (at) {
        const long device = PyLong_AsLong(at.p);
        if (device == -1 && PyErr_Occurred()) return false;
        if (device < 0) return refuse("%s is not on the GPU", name);
        return device == t_device ? true : refuse("%s is on device %ld, the current one is %d", name, device, t_device);
    }
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return false;
    PyErr_Clear();
    Ref cuda(PyObject_GetAttr(t, s_is_cuda));
    if (!cuda) return false;
    const int yes = PyObject_IsTrue(cuda.p);
    if (yes < 0) return false;
    return yes ? true : refuse("%s is not on the GPU", name);
}
bool address(PyObject *t, void **out) {
    Ref p(PyObject_CallMethodNoArgs(t, s_data_ptr));
    if (!p) return false;
    *out = PyLong_AsVoidPtr(p.p);
    return !PyErr_Occurred();
}

struct Matrix { void *p = nullptr; long long ld = 0, rows = 0, cols = 0; int type = OTHER; };
// whether an element type is what is asked for: a code, or -1: fp32, bf16 or fp16
bool fits(int type, int like) { return like < 0 ? type <= B2_F16 : type == like || (like == BYTE && type == INT8); }
// rows, cols: what they have to be (-1: anything); like: the element type it has to have (-1: fp32, bf16 or fp16; BYTE)
bool matrix(PyObject *t, const char *name, long long rows, long long cols, int like, Matrix &m) {
    m = Matrix();
    if (t == Py_None) return true;
    Ref shape(PyObject_GetAttr(t, s_shape));
    if (!shape) return false;
    if (!PyTuple_Check(shape.p) || PyTuple_GET_SIZE(shape.p) != 2) return refuse("%s has the shape %S, not (rows, columns)", name, shape.p);
    m.rows = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.p, 0));
    m.cols = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.p, 1));
    if (PyErr_Occurred()) return false;
    if ((rows >= 0 && m.rows != rows) || (cols >= 0 && m.cols != cols)) return refuse("%s has the shape %S, not (%lld, %lld) (-1: any)", name, shape.p, rows, cols);
    if (!on_gpu(t, name)) return false;
    Ref dtype(PyObject_GetAttr(t, s_dtype));
    m.type = type_of(dtype);
    if (m.type < 0) return false;
    if (!fits(m.type, like)) return refuse("%s has the element type %S", name, dtype.p);
    Ref stride(PyObject_CallMethodNoArgs(t, s_stride));
    if (!stride) return false;
    if (!PyTuple_Check(stride.p) || PyTuple_GET_SIZE(stride.p) != 2) return refuse("%s has the strides %S", name, stride.p);
    const long long ld = PyLong_AsLongLong(PyTuple_GET_ITEM(stride.p, 0)), unit = PyLong_AsLongLong(PyTuple_GET_ITEM(stride.p, 1));
    if (PyErr_Occurred()) return false;
    if ((unit != 1 && m.cols > 1) || (ld < m.cols && m.rows > 1)) return refuse("%s has the strides %S: its rows have to be contiguous and apart", name, stride.p);
    if (m.cols > 0x7fffffff) return refuse("%s has the shape %S: too many columns", name, shape.p);
    m.ld = ld > m.cols ? ld : m.cols;
    return address(t, &m.p);
}
// address of n contiguous elements
bool vector(PyObject *t, const char *name, long long n, int like, void **out) {
    *out = nullptr;
    if (t == Py_None) return true;
    if (!on_gpu(t, name)) return false;
    Ref dtype(PyObject_GetAttr(t, s_dtype));
    const int type = type_of(dtype);
    if (type < 0) return false;
    if (!fits(type, like)) return refuse("%s has the element type %S, not %s", name, dtype.p, like == B2_F32 ? "float32" : like == INT32 ? "int32" : "uint8, int8 or bool");
    Ref count(PyObject_CallMethodNoArgs(t, s_numel)), whole(PyObject_CallMethodNoArgs(t, s_is_contiguous));
    if (!count || !whole) return false;
    const long long have = PyLong_AsLongLong(count.p);
    const int ok = PyObject_IsTrue(whole.p);
    if (PyErr_Occurred()) return false;
    if (have != n || !ok) return refuse("%s has %lld elements%s, not %lld contiguous ones", name, have, ok ? "" : " that are not contiguous", n);
    return address(t, out);
}
bool workspace(PyObject *t, void **p, size_t *bytes) {
    *p = nullptr;
    *bytes = 0;
    if (t == Py_None) return true;
    if (!on_gpu(t, "the workspace")) return false;
    Ref dtype(PyObject_GetAttr(t, s_dtype)), count(PyObject_CallMethodNoArgs(t, s_numel)), whole(PyObject_CallMethodNoArgs(t, s_is_contiguous));
    if (!count || !whole) return false;
    const int type = type_of(dtype);
    if (type < 0) return false;
    const long long n = PyLong_AsLongLong(count.p);
    const int ok = PyObject_IsTrue(whole.p);
    if (PyErr_Occurred()) return false;
    if (!ok || type == OTHER) return refuse("the workspace is not a contiguous tensor of bytes");
    *bytes = (size_t)n * (type == B2_F32 || type == INT32 ? 4 : type == BYTE || type == INT8 ? 1 : 2);
    return address(t, p);
}
bool number(PyObject *o, float *out) { const double v = PyFloat_AsDouble(o); *out = (float)v; return !(v == -1.0 && PyErr_Occurred()); }
bool flag(PyObject *o, int *out) { *out = PyObject_IsTrue(o); return *out >= 0; }
bool stream_of(PyObject *o, b2_stream *out) {
    *out = nullptr;
    if (o == Py_None) return true;
    *out = PyLong_AsVoidPtr(o);
    return !PyErr_Occurred();
}
bool count_of(PyObject *t, const char *name, long long *out) {
    Ref n(PyObject_CallMethodNoArgs(t, s_numel));
    if (!n) { PyErr_Clear(); return refuse("%s is no tensor", name); }
    *out = PyLong_AsLongLong(n.p);
    return !PyErr_Occurred();
}
PyObject *done(int rc) {
    if (!rc) Py_RETURN_NONE;
    refuse("b2lstm error %d: %s", rc, api.last_error());
    return nullptr;
}
// the beginning of every call
bool arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) return refuse("%zd arguments instead of %zd", n, want);
    t_device = api.current_device();
    return true;
}

// a table's rows are an int in the library
bool few_rows(const Matrix &m) { return m.rows <= 0x7fffffff ? true : refuse("a table of %lld rows", m.rows); }

#define CALL(expr)                    \
    int rc;                           \
    Py_BEGIN_ALLOW_THREADS rc = expr; \
    Py_END_ALLOW_THREADS return done(rc)

// out, table, tokens, scale, stream
PyObject *embedding_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix out, table;
    void *tokens;
    long long rows;
    float scale;
    b2_stream st;
    if (!arguments(n, 5) || !count_of(a[2], "tokens", &rows) || !matrix(a[1], "table", -1, -1, -1, table) || !few_rows(table) || !matrix(a[0], "out", rows, table.cols, -1, out) ||
        !vector(a[2], "tokens", rows, INT32, &tokens) || !number(a[3], &scale) || !stream_of(a[4], &st))
        return nullptr;
    CALL(api.embedding_forward(out.p, out.type, out.ld, table.p, table.type, table.ld, (int)table.rows, (int)table.cols, (const int *)tokens, rows, scale, st));
}
// dtable, dout, tokens, scale, accumulate, workspace, stream
PyObject *embedding_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix table, dout;
    void *tokens, *ws;
    size_t bytes;
    long long rows;
    float scale;
    int add;
    b2_stream st;
    if (!arguments(n, 7) || !count_of(a[2], "tokens", &rows) || !matrix(a[0], "dtable", -1, -1, -1, table) || !few_rows(table) || !matrix(a[1], "dout", rows, table.cols, -1, dout) ||
        !vector(a[2], "tokens", rows, INT32, &tokens) || !number(a[3], &scale) || !flag(a[4], &add) || !workspace(a[5], &ws, &bytes) || !stream_of(a[6], &st))
        return nullptr;
    CALL(api.embedding_backward(table.p, table.type, table.ld, (int)table.rows, (int)table.cols, dout.p, dout.type, dout.ld, (const int *)tokens, rows, scale, add, ws, bytes,
                                st));
}

// w_pre, b_pre, w_post, b_post, gate, stats, pat_types, layer_norm, eps, residual_scale (10 arguments from a[0] on); x gives the sizes
bool block_norm(PyObject *const *a, const Matrix &x, b2_block_norm &d) {
    Matrix gate;
    void *v[6];
    if (!vector(a[0], "w_pre", x.cols, B2_F32, &v[0]) || !vector(a[1], "b_pre", x.cols, B2_F32, &v[1]) || !vector(a[2], "w_post", x.cols, B2_F32, &v[2]) ||
        !vector(a[3], "b_post", x.cols, B2_F32, &v[3]) || !matrix(a[4], "gate", -1, x.cols, x.type, gate) || !vector(a[5], "stats", 4 * x.rows, B2_F32, &v[4]) ||
        !vector(a[6], "pat_types", x.rows, BYTE, &v[5]) || !flag(a[7], &d.layer_norm) || !number(a[8], &d.eps) || !number(a[9], &d.residual_scale))
        return false;
    d.type = x.type;
    d.dim = (int)x.cols;
    d.rows = x.rows;
    d.w_pre = (const float *)v[0]; d.b_pre = (const float *)v[1]; d.w_post = (const float *)v[2]; d.b_post = (const float *)v[3];
    d.gate = gate.p; d.gate_rows = gate.rows; d.ld_gate = gate.ld;
    d.stats = (float *)v[4];
    d.pat_types = (const char *)v[5];
    return true;
}
// x, f, y, h, the 10 of block_norm, stream
PyObject *block_norm_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix x, f, y, h;
    b2_block_norm d;
    b2_stream st;
    if (!arguments(n, 15) || !matrix(a[0], "x", -1, -1, -1, x)) return nullptr;
    if (a[0] == Py_None) { refuse("null pointer: x is needed"); return nullptr; }
    if (!block_norm(a + 4, x, d) || !matrix(a[1], "f", x.rows, x.cols, x.type, f) || !matrix(a[2], "y", x.rows, x.cols, x.type, y) ||
        !matrix(a[3], "h", x.rows, x.cols, x.type, h) || !stream_of(a[14], &st))
        return nullptr;
    CALL(api.block_norm_forward(&d, x.p, x.ld, f.p, f.ld, y.p, y.ld, h.p, h.ld, st));
}
// dx, df, dy, dh, y, f, dgate, dw_pre, db_pre, dw_post, db_post, the 10 of block_norm, workspace, stream
PyObject *block_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix m[6], dgate, like;
    static const char *const names[6] = {"dx", "df", "dy", "dh", "y", "f"};
    static const char *const sums[4] = {"dw_pre", "db_pre", "dw_post", "db_post"};
    void *w[4], *ws;
    size_t bytes;
    b2_block_norm d;
    b2_stream st;
    if (!arguments(n, 23)) return nullptr;
    const int given = a[2] != Py_None ? 2 : 3;
    if (a[given] == Py_None) { refuse("dy or dh is needed"); return nullptr; }
    if (a[6] != Py_None && a[15] == Py_None) { refuse("dgate is given without the gate"); return nullptr; }
    if (!matrix(a[given], names[given], -1, -1, -1, like) || !block_norm(a + 11, like, d)) return nullptr;
    for (int i = 0; i < 6; ++i)
        if (!matrix(a[i], names[i], like.rows, like.cols, like.type, m[i])) return nullptr;
    if (!matrix(a[6], "dgate", d.gate_rows, like.cols, like.type, dgate)) return nullptr;
    for (int i = 0; i < 4; ++i)
        if (!vector(a[7 + i], sums[i], like.cols, B2_F32, &w[i])) return nullptr;
    if (!workspace(a[21], &ws, &bytes) || !stream_of(a[22], &st)) return nullptr;
    CALL(api.block_norm_backward(&d, m[0].p, m[0].ld, m[1].p, m[1].ld, dgate.p, dgate.ld, (float *)w[0], (float *)w[1], (float *)w[2], (float *)w[3], m[2].p, m[2].ld, m[3].p,
                                 m[3].ld, m[4].p, m[4].ld, m[5].p, m[5].ld, ws, bytes, st));
}

// a mask of bytes, [vocab] or [rows, vocab]
bool mask_of(PyObject *t, long long rows, long long vocab, Matrix &m) {
    m = Matrix();
    if (t == Py_None) return true;
    Ref shape(PyObject_GetAttr(t, s_shape));
    if (!shape) return false;
    if (PyTuple_Check(shape.p) && PyTuple_GET_SIZE(shape.p) == 1) return vector(t, "mask", vocab, BYTE, &m.p);
    return matrix(t, "mask", rows, vocab, BYTE, m);
}
// logits, tokens, logprob, lse, entropy, top_tokens, top_logprobs, mask, scale, stream
PyObject *logprob_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix x, mask;
    void *tokens, *lp, *lse, *entropy, *top_tokens, *top_lp;
    long long top = 0;
    float scale;
    b2_stream st;
    if (!arguments(n, 10) || !matrix(a[0], "logits", -1, -1, -1, x)) return nullptr;
    if (a[0] == Py_None) { refuse("null pointer: the logits are needed"); return nullptr; }
    if (a[5] != Py_None) {
        Ref shape(PyObject_GetAttr(a[5], s_shape));
        if (!shape) return nullptr;
        if (!PyTuple_Check(shape.p) || PyTuple_GET_SIZE(shape.p) < 1) { refuse("top_tokens has the shape %S", shape.p); return nullptr; }
        top = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.p, PyTuple_GET_SIZE(shape.p) - 1));
        if (PyErr_Occurred()) return nullptr;
        if (top > 1 << 20) top = 1 << 20;
    }
    if (!mask_of(a[7], x.rows, x.cols, mask) || !vector(a[1], "tokens", x.rows, INT32, &tokens) || !vector(a[2], "logprob", x.rows, B2_F32, &lp) ||
        !vector(a[3], "lse", x.rows, B2_F32, &lse) || !vector(a[4], "entropy", x.rows, B2_F32, &entropy) || !vector(a[5], "top_tokens", x.rows * top, INT32, &top_tokens) ||
        !vector(a[6], "top_logprobs", x.rows * top, B2_F32, &top_lp) || !number(a[8], &scale) || !stream_of(a[9], &st))
        return nullptr;
    CALL(api.logprob_forward(x.p, x.type, x.rows, (int)x.cols, x.ld, (const unsigned char *)mask.p, mask.ld, scale, (const int *)tokens, (float *)lp, (float *)lse,
                             (float *)entropy, (int)top, (int *)top_tokens, (float *)top_lp, st));
}
// dlogits, logits, tokens, lse, dlogprob, entropy, dentropy, mask, scale, stream
PyObject *logprob_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix d, x, mask;
    void *tokens, *lse, *g, *entropy, *h;
    float scale;
    b2_stream st;
    if (!arguments(n, 10) || !matrix(a[1], "logits", -1, -1, -1, x)) return nullptr;
    if (a[1] == Py_None) { refuse("null pointer: the logits are needed"); return nullptr; }
    if (!matrix(a[0], "dlogits", x.rows, x.cols, x.type, d) || !mask_of(a[7], x.rows, x.cols, mask) || !vector(a[2], "tokens", x.rows, INT32, &tokens) ||
        !vector(a[3], "lse", x.rows, B2_F32, &lse) || !vector(a[4], "dlogprob", x.rows, B2_F32, &g) || !vector(a[5], "entropy", x.rows, B2_F32, &entropy) ||
        !vector(a[6], "dentropy", x.rows, B2_F32, &h) || !number(a[8], &scale) || !stream_of(a[9], &st))
        return nullptr;
    CALL(api.logprob_backward(d.p, d.ld, x.p, x.type, x.rows, (int)x.cols, x.ld, (const unsigned char *)mask.p, mask.ld, scale, (const int *)tokens, (const float *)lse,
                              (const float *)g, (const float *)entropy, (const float *)h, st));
}

// a list's tensors, all on one device (-1: not known)
bool list_on_gpu(PyObject *device) {
    const long d = PyLong_AsLong(device);
    if (d == -1 && PyErr_Occurred()) return false;
    return d < 0 || d == t_device ? true : refuse("the tensors are on device %ld, the current one is %d", d, t_device);
}
// address of the list, its length, its device, norm, workspace, stream
PyObject *gradient_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    void *norm, *ws;
    size_t bytes;
    b2_stream st;
    if (!arguments(n, 6)) return nullptr;
    const b2_tensor *list = (const b2_tensor *)PyLong_AsVoidPtr(a[0]);
    const int len = (int)PyLong_AsLong(a[1]);
    if (PyErr_Occurred() || !list_on_gpu(a[2]) || !vector(a[3], "norm", 1, B2_F32, &norm) || !workspace(a[4], &ws, &bytes) || !stream_of(a[5], &st)) return nullptr;
    CALL(api.gradient_norm(list, len, (float *)norm, ws, bytes, st));
}
// address of the list, of the outputs' (0: in place), length, device, max_norm, norm, workspace, stream
PyObject *gradient_clip(PyObject *, PyObject *const *a, Py_ssize_t n) {
    void *norm, *ws;
    size_t bytes;
    float most;
    b2_stream st;
    if (!arguments(n, 8)) return nullptr;
    const b2_tensor *list = (const b2_tensor *)PyLong_AsVoidPtr(a[0]), *out = (const b2_tensor *)PyLong_AsVoidPtr(a[1]);
    const int len = (int)PyLong_AsLong(a[2]);
    if (PyErr_Occurred() || !list_on_gpu(a[3]) || !number(a[4], &most) || !vector(a[5], "norm", 1, B2_F32, &norm) || !workspace(a[6], &ws, &bytes) || !stream_of(a[7], &st)) return nullptr;
    CALL(api.gradient_clip(list, out, len, most, (float *)norm, ws, bytes, st));
}

// the columns of a list [rows, top] that is not None
bool width_of(PyObject *t, const char *name, long long *out) {
    Ref shape(PyObject_GetAttr(t, s_shape));
    if (!shape) return false;
    if (!PyTuple_Check(shape.p) || PyTuple_GET_SIZE(shape.p) != 2) return refuse("%s has the shape %S, not (rows, columns)", name, shape.p);
    *out = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.p, 1));
    if (PyErr_Occurred()) return false;
    if (*out > 1 << 20) *out = 1 << 20;
    return true;
}
// logits, top_tokens, top_logprobs, loss, lse, lse_rest, scale, stream
PyObject *distill_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix x;
    void *tokens, *lp, *loss, *lse, *rest;
    long long top;
    float scale;
    b2_stream st;
    if (!arguments(n, 8) || !matrix(a[0], "logits", -1, -1, -1, x)) return nullptr;
    for (int i = 0; i < 5; ++i)
        if (a[i] == Py_None) { refuse("null pointer: all but lse_rest are needed"); return nullptr; }
    if (!width_of(a[1], "top_tokens", &top) || !vector(a[1], "top_tokens", x.rows * top, INT32, &tokens) || !vector(a[2], "top_logprobs", x.rows * top, B2_F32, &lp) ||
        !vector(a[3], "loss", x.rows, B2_F32, &loss) || !vector(a[4], "lse", x.rows, B2_F32, &lse) || !vector(a[5], "lse_rest", x.rows, B2_F32, &rest) ||
        !number(a[6], &scale) || !stream_of(a[7], &st))
        return nullptr;
    CALL(api.distill_forward(x.p, x.type, x.rows, (int)x.cols, x.ld, scale, (const int *)tokens, (const float *)lp, (int)top, (float *)loss, (float *)lse, (float *)rest, st));
}
// dlogits, logits, top_tokens, top_logprobs, lse, lse_rest, dloss, scale, accumulate, stream
PyObject *distill_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix d, x;
    void *tokens, *lp, *lse, *rest, *g;
    long long top;
    float scale;
    int add;
    b2_stream st;
    if (!arguments(n, 10) || !matrix(a[1], "logits", -1, -1, -1, x)) return nullptr;
    for (int i = 0; i < 7; ++i)
        if (i != 5 && a[i] == Py_None) { refuse("null pointer: all but lse_rest are needed"); return nullptr; }
    if (!matrix(a[0], "dlogits", x.rows, x.cols, x.type, d) || !width_of(a[2], "top_tokens", &top) || !vector(a[2], "top_tokens", x.rows * top, INT32, &tokens) ||
        !vector(a[3], "top_logprobs", x.rows * top, B2_F32, &lp) || !vector(a[4], "lse", x.rows, B2_F32, &lse) || !vector(a[5], "lse_rest", x.rows, B2_F32, &rest) ||
        !vector(a[6], "dloss", x.rows, B2_F32, &g) || !number(a[7], &scale) || !flag(a[8], &add) || !stream_of(a[9], &st))
        return nullptr;
    CALL(api.distill_backward(d.p, d.ld, x.p, x.type, x.rows, (int)x.cols, x.ld, scale, (const int *)tokens, (const float *)lp, (int)top, (const float *)lse,
                              (const float *)rest, (const float *)g, add, st));
}
// logits, scores, top_scores, top_beams, top_tokens, finished, weights, end_token, mask, scale, workspace, stream
PyObject *beam_select(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix x, mask;
    void *scores, *best, *from, *tokens, *finished, *weights, *ws;
    size_t bytes;
    long long top, groups;
    float scale;
    b2_stream st;
    if (!arguments(n, 12) || !matrix(a[0], "logits", -1, -1, -1, x)) return nullptr;
    for (int i = 0; i < 5; ++i)
        if (a[i] == Py_None) { refuse("null pointer: logits, scores and results are needed"); return nullptr; }
    if (!width_of(a[2], "top_scores", &top) || !count_of(a[2], "top_scores", &groups)) return nullptr;
    groups = top > 0 ? groups / top : 0;
    if (groups < 1 ? x.rows > 0 : x.rows % groups != 0) { refuse("%lld rows of logits for %lld sequences", x.rows, groups); return nullptr; }
    const long long beams = groups ? x.rows / groups : 1;
    const long end = PyLong_AsLong(a[7]);
    if (PyErr_Occurred()) return nullptr;
    if (beams > 1 << 20 || end != (int)end) { refuse("%lld beams a sequence, end_token %ld", beams, end); return nullptr; }
    if (!mask_of(a[8], x.rows, x.cols, mask) || !vector(a[1], "scores", x.rows, B2_F32, &scores) || !vector(a[2], "top_scores", groups * top, B2_F32, &best) ||
        !vector(a[3], "top_beams", groups * top, INT32, &from) || !vector(a[4], "top_tokens", groups * top, INT32, &tokens) ||
        !vector(a[5], "finished", x.rows, BYTE, &finished) || !vector(a[6], "weights", x.rows, B2_F32, &weights) || !number(a[9], &scale) ||
        !workspace(a[10], &ws, &bytes) || !stream_of(a[11], &st))
        return nullptr;
    CALL(api.beam_select(x.p, x.type, groups, (int)beams, (int)x.cols, x.ld, (const unsigned char *)mask.p, mask.ld, scale, (const float *)scores,
                         (const unsigned char *)finished, (const float *)weights, (int)end, (int)top, (float *)best, (int *)from, (int *)tokens, ws, bytes, st));
}
// address of the list, its length, its device, its beams (-1: an empty list), parents, stream
PyObject *beam_reorder(PyObject *, PyObject *const *a, Py_ssize_t n) {
    void *parents;
    long long count, beams;
    b2_stream st;
    if (!arguments(n, 6)) return nullptr;
    const b2_state *list = (const b2_state *)PyLong_AsVoidPtr(a[0]);
    const int len = (int)PyLong_AsLong(a[1]);
    const long long rows = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred() || !list_on_gpu(a[2]) || !width_of(a[4], "parents", &beams) || !count_of(a[4], "parents", &count) ||
        !vector(a[4], "parents", count, INT32, &parents) || !stream_of(a[5], &st))
        return nullptr;
    if (rows >= 0 && count != rows) { refuse("%lld parents for %lld beams", count, rows); return nullptr; }
    CALL(api.beam_reorder(list, len, (const int *)parents, beams > 0 ? count / beams : 0, (int)beams, st));
}
// q, scales, x, stream
PyObject *int8_quantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix q, x;
    void *scales;
    b2_stream st;
    if (!arguments(n, 4)) return nullptr;
    for (int i = 0; i < 3; ++i)
        if (a[i] == Py_None) { refuse("null pointer: q, scales and x are needed"); return nullptr; }
    if (!matrix(a[2], "x", -1, -1, -1, x) || !matrix(a[0], "q", x.rows, x.cols, INT8, q) || !vector(a[1], "scales", x.rows, B2_F32, &scales) || !stream_of(a[3], &st)) return nullptr;
    CALL(api.int8_quantize((signed char *)q.p, q.ld, (float *)scales, x.p, x.type, x.rows, (int)x.cols, x.ld, st));
}
// out, x, x_scales, w, w_scales, bias, workspace, stream
PyObject *int8_product(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Matrix out, x, w;
    void *xs, *wsc, *bias, *ws;
    size_t bytes;
    b2_stream st;
    if (!arguments(n, 8)) return nullptr;
    for (int i = 0; i < 5; ++i)
        if (i != 2 && a[i] == Py_None) { refuse("null pointer: out, x, w and w_scales are needed"); return nullptr; }
    const bool given = a[2] != Py_None;
    if (!matrix(a[3], "w", -1, -1, INT8, w)) return nullptr;
    if (w.rows > 0x7fffffff) { refuse("w has %lld channels", w.rows); return nullptr; }
    if (!matrix(a[1], "x", -1, w.cols, given ? INT8 : -1, x) || !matrix(a[0], "out", x.rows, w.rows, -1, out) || !vector(a[2], "x_scales", x.rows, B2_F32, &xs) ||
        !vector(a[4], "w_scales", w.rows, B2_F32, &wsc) || !vector(a[5], "bias", w.rows, B2_F32, &bias) || !workspace(a[6], &ws, &bytes) || !stream_of(a[7], &st))
        return nullptr;
    CALL(api.int8_product(out.p, out.type, out.ld, x.p, given ? (int)B2_I8 : x.type, x.ld, (const float *)xs, (const signed char *)w.p, w.ld, (const float *)wsc,
                          (const float *)bias, x.rows, (int)w.rows, (int)w.cols, ws, bytes, st));
}

// bind({name: address}, B2Error)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 2) { refuse("%zd arguments instead of 2", n); return nullptr; }
    const struct { const char *name; void **to; } all[] = {
        {"b2_last_error_string", (void **)&api.last_error}, {"b2_current_device", (void **)&api.current_device}, {"b2_embedding_forward", (void **)&api.embedding_forward},
        {"b2_embedding_backward", (void **)&api.embedding_backward}, {"b2_block_norm_forward", (void **)&api.block_norm_forward},
        {"b2_block_norm_backward", (void **)&api.block_norm_backward}, {"b2_logprob_forward", (void **)&api.logprob_forward},
        {"b2_logprob_backward", (void **)&api.logprob_backward}, {"b2_gradient_norm", (void **)&api.gradient_norm}, {"b2_gradient_clip", (void **)&api.gradient_clip},
        {"b2_distill_forward", (void **)&api.distill_forward}, {"b2_distill_backward", (void **)&api.distill_backward}, {"b2_beam_select", (void **)&api.beam_select},
        {"b2_beam_reorder", (void **)&api.beam_reorder}, {"b2_int8_quantize", (void **)&api.int8_quantize}, {"b2_int8_product", (void **)&api.int8_product}};
    for (const auto &f : all) {
        PyObject *p = PyDict_GetItemString(a[0], f.name);
        if (!p) { refuse("%s is missing", f.name); return nullptr; }
        *f.to = PyLong_AsVoidPtr(p);
        if (PyErr_Occurred()) return nullptr;
    }
    Py_INCREF(a[1]);
    Py_XDECREF(g_error);
    g_error = a[1];
    Py_RETURN_NONE;
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(embedding_forward), METHOD(embedding_backward), METHOD(block_norm_forward), METHOD(block_norm_backward),
                         METHOD(logprob_forward), METHOD(logprob_backward), METHOD(gradient_norm), METHOD(gradient_clip),
                         METHOD(distill_forward), METHOD(distill_backward), METHOD(beam_select), METHOD(beam_reorder), METHOD(int8_quantize), METHOD(int8_product), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", "tensor side of the token operators' binding", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) {
    const struct { PyObject **to; const char *text; } names[] = {{&s_shape, "shape"}, {&s_stride, "stride"}, {&s_dtype, "dtype"}, {&s_is_cuda, "is_cuda"}, {&s_get_device, "get_device"},
                                                                 {&s_data_ptr, "data_ptr"}, {&s_numel, "numel"}, {&s_is_contiguous, "is_contiguous"}};
    for (const auto &n : names)
        if (!(*n.to = PyUnicode_InternFromString(n.text))) return nullptr;
    if (!(g_types = PyDict_New())) return nullptr;
    return PyModule_Create(&module);
}
