// Host side of the tensor-level serving calls (ecog2txt_amd/serving.py): argument checks, outputs, workspaces and the call into
// libecog2txt_hip.so, as a CPython extension on torch's C++ tensors.  The operators' small calls take 3 to 8 us on the GPU; checks, outputs
// and ctypes from Python took 11 us a call, this takes 5 (the launch among them).
// The library's functions come as addresses (bind), from the library that hip_lib.py has loaded: this file links against torch only.
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include "ecog2txt_hip.h"

namespace {
#define E2T_BOUND(X) X(e2t_quant_rows_i8) X(e2t_gemm_nt_i8) X(e2t_linear_i8_ws_bytes) X(e2t_linear_i8) X(e2t_sample_ws_bytes) X(e2t_sample_rows) X(e2t_last_error)
#define X(f) decltype(&::f) f##_p = nullptr;
E2T_BOUND(X)
#undef X
PyObject *raw_stream, *s_q, *s_scale, *s_cols, *rows_type;        // torch's current-stream function; attribute names and class of Int8Rows

struct Bad {};                                             // (the Python error is set)
[[noreturn]] void bad(const char* f, ...) {
    va_list ap;
    va_start(ap, f);
    char what[256];
    vsnprintf(what, sizeof what, f, ap);
    va_end(ap);
    PyErr_Format(PyExc_ValueError, "ecog2txt_amd.serving: %s", what);
    throw Bad();
}
const char* type_name(at::ScalarType t) { return t == at::kFloat ? "float32" : t == at::kInt ? "int32" : t == at::kChar ? "int8" : "bfloat16"; }

// nothing here has a gradient: a tensor that asks for one, in reverse or in forward mode, is refused; and memory is read as it lies, so
// that a view which stands for its negative (the imaginary part of a conjugate) is refused, too
void plain(const at::Tensor& t, const char* name) {
    if (t.is_neg()) bad("%s is a view of the negative of what its memory holds (use its resolve_neg())", name);
    if (!t.unsafeGetTensorImpl()->autograd_meta()) return;       // (most have none: spares three calls into torch)
    if (t.requires_grad() && at::GradMode::is_enabled()) bad("%s asks for a gradient: the serving operators have none (use torch.no_grad())", name);
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        bad("%s has a forward-mode tangent: the serving operators pass none on", name);
}
struct Mat { const at::Tensor* t; int64_t rows, cols, ld; int dev; };
// a 2-D device tensor with contiguous rows
Mat matrix(PyObject* o, const char* name, at::ScalarType t0, at::ScalarType t1) {
    const bool is = THPVariable_Check(o);
    if (is) plain(THPVariable_Unpack(o), name);
    if (!is || !THPVariable_Unpack(o).is_cuda() || THPVariable_Unpack(o).dim() != 2 || (THPVariable_Unpack(o).scalar_type() != t0 && THPVariable_Unpack(o).scalar_type() != t1))
        bad("%s must be a 2-D device tensor of %s%s%s", name, type_name(t0), t0 != t1 ? " / " : "", t0 != t1 ? type_name(t1) : "");
    const at::Tensor& t = THPVariable_Unpack(o);
    Mat m{&t, t.size(0), t.size(1), t.stride(0), t.get_device()};
    if (m.cols == 0) bad("%s has no columns", name);
    if (t.stride(1) != 1 && m.cols > 1) bad("%s must have contiguous rows (stride 1 along the last dimension)", name);
    if (m.ld < m.cols) { if (m.rows > 1) bad("rows of %s overlap", name); m.ld = m.cols; }
    if (m.rows > E2T_I8_MAX_ROWS || m.cols > E2T_I8_MAX_ROWS) bad("%s is too large", name);
    return m;
}
void* vector(PyObject* o, int64_t n, at::ScalarType type, int dev, const char* name) {
    if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        plain(t, name);
        if (t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && t.dim() == 1 && t.size(0) == n && t.is_contiguous()) return t.data_ptr();
    }
    bad("%s must be a contiguous %s tensor of %lld on device %d", name, type_name(type), (long long)n, dev);
}
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) { return at::empty(size, like.options().dtype(type).requires_grad(false)); }
void* stream_of(int dev) {
    PyObject* i = PyLong_FromLong(dev);
    PyObject* s = i ? PyObject_CallOneArg(raw_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!s) throw Bad();
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    return p;
}
// f(args ..., the current stream of the device) with the device current
template <class F, class... A> void call(const char* name, int dev, F f, A... a) {
    void* st = stream_of(dev);
    int rc;
    {
        c10::DeviceGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)dev));
        Py_BEGIN_ALLOW_THREADS
        rc = f(a..., st);
        Py_END_ALLOW_THREADS
    }
    if (rc) { PyErr_Format(PyExc_RuntimeError, "%s failed (%d): %s", name, rc, e2t_last_error_p()); throw Bad(); }
}

// a matrix in 8 bits with `cols` columns
struct RowsMem { const at::Tensor* t; int64_t n, ld; int dev; const int8_t* q; const float* scale; };
RowsMem rows_mem(PyObject* q, PyObject* scale, int64_t cols) {
    const Mat m = matrix(q, "q", at::kChar, at::kChar);
    const int64_t cols64 = cols > E2T_I8_MAX_ROWS ? cols : (cols + 63) / 64 * 64;
    if (cols <= 0 || cols64 > m.cols) bad("q needs %lld columns (the %lld of the matrix, rounded up to 64)", (long long)cols64, (long long)cols);
    if (cols > E2T_I8_MAX_K) bad("more than %d columns overflow the 32-bit sums", E2T_I8_MAX_K);
    RowsMem r{m.t, m.rows, m.rows <= 1 ? cols64 : m.ld, m.dev, (const int8_t*)m.t->data_ptr(), nullptr};
    if (r.ld > E2T_I8_MAX_LD) bad("rows of q lie more than %d bytes apart", E2T_I8_MAX_LD);
    if (((uintptr_t)r.q | (uintptr_t)r.ld) & 15) bad("the rows of q must start on 16-byte boundaries");
    r.scale = (const float*)vector(scale, m.rows, at::kFloat, m.dev, "scale");
    return r;
}
// an Int8Rows, by its attributes, which may have been set (or their tensors resized) since it was made: they are checked in every call
struct Rows : RowsMem {
    THPObjectPtr hold_q, hold_scale;
    int64_t cols = 0;
    explicit Rows(PyObject* o, const char* name) {
        const int is = PyObject_IsInstance(o, rows_type);
        if (is < 0) throw Bad();
        if (!is) bad("%s must be Int8Rows", name);
        THPObjectPtr c(PyObject_GetAttr(o, s_cols));
        hold_q = PyObject_GetAttr(o, s_q); hold_scale = PyObject_GetAttr(o, s_scale);
        if (!c || !hold_q || !hold_scale) throw Bad();
        cols = PyLong_AsLongLong(c.get());
        if (cols == -1 && PyErr_Occurred()) throw Bad();
        *(RowsMem*)this = rows_mem(hold_q.get(), hold_scale.get(), cols);
    }
};
struct Out { at::Tensor made; const at::Tensor* t; int64_t n, ld; const float* bias; int flags; };
// weights, bias, output type and output of a product with `rows` rows of activations
Out output(const Rows& w, int64_t cols, PyObject* bias, PyObject* out_dtype, PyObject* relu, PyObject* out, int64_t rows, const at::Tensor& like) {
    const int dev = like.get_device();
    if (w.dev != dev) bad("the weights must be Int8Rows on device %d", dev);
    if (w.cols != cols) bad("%lld columns of activations, %lld of weights", (long long)cols, (long long)w.cols);
    Out o{};
    o.n = w.n;
    if (o.n == 0) bad("the weights have no rows");
    const at::ScalarType type = THPDtype_Check(out_dtype) ? ((THPDtype*)out_dtype)->scalar_type : at::kByte;
    if (type != at::kFloat && type != at::kBFloat16) bad("out_dtype must be float32 or bfloat16");
    o.bias = bias == Py_None ? nullptr : (const float*)vector(bias, o.n, at::kFloat, dev, "bias");
    const int r = PyObject_IsTrue(relu);
    if (r < 0) throw Bad();
    o.flags = (r ? E2T_GEMM_RELU : 0) | (type == at::kBFloat16 ? E2T_GEMM_OUT_BF16 : 0);
    if (out == Py_None) { o.made = fresh(like, {rows, o.n}, type); o.t = &o.made; o.ld = o.n; return o; }
    const Mat m = matrix(out, "out", type, type);
    if (m.dev != dev || m.rows != rows || m.cols != o.n) bad("out must be (%lld, %lld) on device %d", (long long)rows, (long long)o.n, dev);
    o.t = m.t; o.ld = m.ld;
    return o;
}
int dt_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? E2T_DT_BF16 : E2T_DT_F32; }
PyObject* wrap(const Out& o, PyObject* out) {
    if (out == Py_None) return THPVariable_Wrap(o.made);
    if (!o.t->is_inference()) o.t->unsafeGetTensorImpl()->bump_version();       // (a graph that saved its old values notices)
    Py_INCREF(out);
    return out;
}

PyObject* bind(PyObject*, PyObject* const*, Py_ssize_t);
// every entry: C++ exceptions become Python's
#define E2T_PY(name, n)                                                                         \
    PyObject* name##_(PyObject* const* a);                                                       \
    PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t given) {                            \
        HANDLE_TH_ERRORS                                                                         \
        if (!rows_type && name != bind) { PyErr_SetString(PyExc_RuntimeError, "_serving_host: not bound"); return nullptr; } \
        if (given != n) { PyErr_SetString(PyExc_TypeError, #name ": " #n " arguments"); return nullptr; } \
        try { return name##_(a); } catch (const Bad&) { return nullptr; }                         \
        END_HANDLE_TH_ERRORS                                                                     \
    }                                                                                            \
    PyObject* name##_(PyObject* const* a)

// check_rows(q, scale, cols) -> row stride
E2T_PY(check_rows, 3) {
    const int64_t cols = PyLong_AsLongLong(a[2]);
    if (cols == -1 && PyErr_Occurred()) throw Bad();
    return PyLong_FromLongLong(rows_mem(a[0], a[1], cols).ld);
}
// quantize(x) -> q, scale
E2T_PY(quantize, 1) {
    const Mat x = matrix(a[0], "x", at::kFloat, at::kBFloat16);
    if (x.cols > E2T_I8_MAX_K) bad("more than %d columns overflow the 32-bit sums", E2T_I8_MAX_K);
    const at::Tensor q = fresh(*x.t, {x.rows, (x.cols + 63) / 64 * 64}, at::kChar), scale = fresh(*x.t, {x.rows}, at::kFloat);
    if (x.rows)
        call("e2t_quant_rows_i8", x.dev, e2t_quant_rows_i8_p, x.t->data_ptr(), dt_of(*x.t), (long long)x.ld, (int)x.rows, (int)x.cols, (int8_t*)q.data_ptr(),
             (long long)q.size(1), (float*)scale.data_ptr());
    return Py_BuildValue("NN", THPVariable_Wrap(q), THPVariable_Wrap(scale));
}
// matmul(a, w, bias, out_dtype, relu, out) -> out
E2T_PY(matmul, 6) {
    const Rows x(a[0], "a"), w(a[1], "w");
    const Out o = output(w, x.cols, a[2], a[3], a[4], a[5], x.n, *x.t);
    if (x.n)
        call("e2t_gemm_nt_i8", x.dev, e2t_gemm_nt_i8_p, x.q, (long long)x.ld, x.scale, w.q, (long long)w.ld, w.scale, o.bias, o.t->data_ptr(), (long long)o.ld, (int)x.n,
             (int)o.n, (int)x.cols, o.flags);
    return wrap(o, a[5]);
}
// linear(x, w, bias, out_dtype, relu, out) -> out
E2T_PY(linear, 6) {
    const Mat x = matrix(a[0], "x", at::kFloat, at::kBFloat16);
    const Rows w(a[1], "w");
    const Out o = output(w, x.cols, a[2], a[3], a[4], a[5], x.rows, *x.t);
    if (x.rows) {
        const size_t need = e2t_linear_i8_ws_bytes_p((int)x.rows, (int)o.n, (int)x.cols);
        at::Tensor ws;
        if (need) ws = fresh(*x.t, {(int64_t)need}, at::kByte);
        call("e2t_linear_i8", x.dev, e2t_linear_i8_p, x.t->data_ptr(), dt_of(*x.t), (long long)x.ld, w.q, (long long)w.ld, w.scale, o.bias,
             o.t->data_ptr(), (long long)o.ld, (int)x.rows, (int)o.n, (int)x.cols, o.flags, need ? ws.data_ptr() : nullptr, need);
    }
    return wrap(o, a[5]);
}
// sample(logits, u, temperature, top_k, top_p, min_p) -> token, logprob
E2T_PY(sample, 6) {
    const Mat l = matrix(a[0], "logits", at::kFloat, at::kBFloat16);
    if (l.cols > E2T_SAMPLE_MAX_V) bad("more than %d logits a row", E2T_SAMPLE_MAX_V);
    const float* u = (const float*)vector(a[1], l.rows, at::kFloat, l.dev, "u");
    e2t_sample_cfg c{};
    auto number = [&](PyObject* v, const char* name, float& all, const float*& rows) {
        if (THPVariable_Check(v)) { rows = (const float*)vector(v, l.rows, at::kFloat, l.dev, name); return; }
        all = (float)PyFloat_AsDouble(v);
        if (PyErr_Occurred()) throw Bad();
    };
    number(a[2], "temperature", c.temperature, c.temperature_rows);
    number(a[4], "top_p", c.top_p, c.top_p_rows);
    number(a[5], "min_p", c.min_p, c.min_p_rows);
    if (THPVariable_Check(a[3])) c.top_k_rows = (const int32_t*)vector(a[3], l.rows, at::kInt, l.dev, "top_k");
    else {
        PyObject* k = PyNumber_Long(a[3]);
        int over = 0;
        const long long v = k ? PyLong_AsLongLongAndOverflow(k, &over) : 0;
        Py_XDECREF(k);
        if (PyErr_Occurred()) throw Bad();
        c.top_k = over > 0 || v > 0x7FFFFFFF ? 0x7FFFFFFF : over < 0 || v < 0 ? 0 : (int)v;
    }
    const at::Tensor token = fresh(*l.t, {l.rows}, at::kInt), logprob = fresh(*l.t, {l.rows}, at::kFloat);
    if (l.rows) {
        const size_t need = e2t_sample_ws_bytes_p((int)l.rows, (int)l.cols);
        at::Tensor ws;
        if (need) ws = fresh(*l.t, {(int64_t)need}, at::kByte);
        call("e2t_sample_rows", l.dev, e2t_sample_rows_p, l.t->data_ptr(), dt_of(*l.t), (long long)l.ld, (int)l.rows, (int)l.cols, u, (const e2t_sample_cfg*)&c,
             (int32_t*)token.data_ptr(), (float*)logprob.data_ptr(), need ? ws.data_ptr() : nullptr, need);
    }
    return Py_BuildValue("NN", THPVariable_Wrap(token), THPVariable_Wrap(logprob));
}
// bind({name: address}, current-stream function, Int8Rows)
E2T_PY(bind, 3) {
#define X(f)                                                                                        \
    {                                                                                               \
        PyObject* v = PyDict_GetItemString(a[0], #f);                                                \
        f##_p = v ? (decltype(f##_p))PyLong_AsVoidPtr(v) : nullptr;                                  \
        if (!f##_p) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #f); throw Bad(); }     \
    }
    E2T_BOUND(X)
#undef X
    Py_INCREF(a[1]); Py_XSETREF(raw_stream, a[1]);
    Py_INCREF(a[2]); Py_XSETREF(rows_type, a[2]);
    Py_RETURN_NONE;
}
#define E2T_METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {E2T_METHOD(bind), E2T_METHOD(check_rows), E2T_METHOD(quantize), E2T_METHOD(matmul), E2T_METHOD(linear), E2T_METHOD(sample), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__serving_host() {
    s_q = PyUnicode_InternFromString("q"); s_scale = PyUnicode_InternFromString("scale");
    s_cols = PyUnicode_InternFromString("cols");
    return s_q && s_scale && s_cols ? PyModule_Create(&module) : nullptr;
}
