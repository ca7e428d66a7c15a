// row_ops.cpp -- the host side of the row operators (grad_norm.hip, rms_norm.hip, f8.hip): argument
// checks, output allocation and the calls into liblcf's C ABI, as a CPython module over torch's C++
// tensors.  These operators are called on one row as often as on many, and then the host's time is
// all there is: the same checks in Python took 15 to 40 us a call, and 80 us for a list of 78
// gradients.  The library's functions are handed over by address (objectdetection_amd/_lib.py loads
// it), so there is one liblcf in a process and nothing is linked against.
// Every function takes the raw stream last and expects the tensors' device to be the current one.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>

#include "../../../include/lcf.h"

namespace {

struct Err {
    PyObject *type;
    std::string what;
};
[[noreturn]] void fail(PyObject *type, std::string what) { throw Err{type, std::move(what)}; }

#define LCF_FUNCTIONS(F)                                                                                       \
    F(strerror) F(grad_norm_workspace_bytes) F(grad_norm) F(grad_clip) F(rms_norm_fwd) F(rms_norm_workspace_bytes) \
    F(rms_norm_bwd) F(f8_quant) F(f8_gemm_workspace_bytes) F(f8_gemm) F(f8_linear) F(sum_parts)
struct Lib {
#define F(name) decltype(&lcf_##name) name;
    LCF_FUNCTIONS(F)
#undef F
} L;

void check(int rc)
{
    if (rc != LCF_OK) fail(PyExc_RuntimeError, L.strerror(rc));
}

// ---- arguments
const at::Tensor *maybe(PyObject *o)
{
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
    return &THPVariable_Unpack(o);
}
const at::Tensor &need(PyObject *o)
{
    const at::Tensor *t = maybe(o);
    if (!t) fail(PyExc_TypeError, "expected a tensor, got None");
    return *t;
}
long long number(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        fail(PyExc_TypeError, "expected a whole number");
    }
    return v;
}
bool truth(PyObject *o) { return PyObject_IsTrue(o) == 1; }
double real(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        fail(PyExc_TypeError, "expected a number");
    }
    return v;
}
void *stream_of(PyObject *o) { return PyLong_AsVoidPtr(o); }

int type_code(at::ScalarType t)
{
    return t == at::kFloat ? LCF_F32 : t == at::kBFloat16 ? LCF_BF16 : t == at::kHalf ? LCF_F16 : -1;
}
at::ScalarType type_of(int code) { return code == LCF_F32 ? at::kFloat : code == LCF_BF16 ? at::kBFloat16 : at::kHalf; }
int f8_code(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? LCF_E4M3 : t == at::kFloat8_e5m2 ? LCF_E5M2 : -1; }
at::ScalarType f8_of(int code) { return code == LCF_E4M3 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2; }

void on_gpu(const at::Tensor &t)
{
    if (!t.is_cuda())
        fail(PyExc_RuntimeError, "objectdetection_amd ops run on the GPU only (no CPU fallback); got a " +
                                     t.device().str() + " tensor");
}
void beside(const at::Tensor &t, const at::Tensor &x, const char *who)
{
    on_gpu(t);
    if (t.get_device() != x.get_device())
        fail(PyExc_RuntimeError, std::string(who) + ": all tensors must be on one device");
}
std::string shape(const at::Tensor &t)
{
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

PyObject *wrap(const at::Tensor &t)
{
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
template <typename... T> PyObject *tuple(const T &...t)
{
    PyObject *items[] = {wrap(t)...};
    PyObject *r = PyTuple_New(sizeof...(t));
    bool bad = !r;
    for (size_t i = 0; i < sizeof...(t); ++i) bad |= !items[i];
    if (bad) {
        for (PyObject *p : items) Py_XDECREF(p);
        Py_XDECREF(r);
        return nullptr;
    }
    for (size_t i = 0; i < sizeof...(t); ++i) PyTuple_SET_ITEM(r, i, items[i]);
    return r;
}

// ---- rows: [..., width] as a matrix with unit stride in a row, copied only where it is not one
struct Rows {
    at::Tensor t;
    long long n, ld;
    void *ptr() const { return t.data_ptr(); }
};
Rows rows_of(const at::Tensor &x, long long width)
{
    if (x.is_contiguous()) return {x, width ? (long long)x.numel() / width : (x.dim() ? (long long)x.size(0) : 0), width};
    at::Tensor v = x.dim() == 2 ? x : x.reshape({-1, width});
    if ((width > 1 && v.stride(1) != 1) || (v.size(0) > 1 && v.stride(0) < width)) v = v.contiguous();
    return {v, (long long)v.size(0), v.size(0) > 1 ? (long long)v.stride(0) : width};
}
int count(long long n, const char *who)
{
    if (n >= 1ll << 31) fail(PyExc_ValueError, std::string(who) + ": fewer than 2^31 rows and columns");
    return (int)n;
}
at::Tensor bytes(size_t n, const at::Tensor &like) { return at::empty({(int64_t)(n < 256 ? 256 : n)}, like.options().dtype(at::kByte)); }

// ---- 8-bit form
struct F8 {
    at::Tensor data, scale;
    long long R = 0, C = 0, ld = 16, lds = 4;
    bool square = false;
    int fmt = 0;
    void *q() const { return data.data_ptr(); }
    unsigned char *s() const { return (unsigned char *)scale.data_ptr(); }
};
F8 f8_empty(long long R, long long C, bool square, int fmt, const at::Tensor &like)
{
    F8 m;
    m.R = R;
    m.C = C;
    m.square = square;
    m.fmt = fmt;
    m.ld = (C + 15) / 16 * 16;
    const long long nb = (C + 127) / 128, sr = square ? (R + 127) / 128 : R;
    m.lds = (nb + 3) / 4 * 4;
    m.data = at::empty({R, m.ld}, like.options().dtype(f8_of(fmt)));
    m.scale = at::empty({sr, m.lds}, like.options().dtype(at::kFloat8_e8m0fnu));
    if (m.ld != C) m.data = m.data.narrow(1, 0, C);
    if (m.lds != nb) m.scale = m.scale.narrow(1, 0, nb);
    return m;
}

// every row on a `to`-byte border and readable up to the next one: as it is, or copied once
at::Tensor bordered(const at::Tensor &t, long long to, long long &ld)
{
    const long long R = t.size(0), C = t.size(1), room = (C + to - 1) / to * to;
    ld = R > 1 ? (long long)t.stride(0) : room;
    if (t.numel() == 0) {
        ld = room ? room : to;
        return t;
    }
    if ((t.stride(1) == 1 || C == 1) && ld >= room && ld % to == 0 && (uintptr_t)t.data_ptr() % to == 0 &&
        (room == C || (long long)t.storage().nbytes() >= t.storage_offset() + (R - 1) * ld + room))
        return t;
    at::Tensor out = at::zeros({R, room}, t.options().dtype(at::kByte));
    out.narrow(1, 0, C).copy_(t.view(at::kByte));
    ld = room;
    return out.view(t.scalar_type()).narrow(1, 0, C);
}

F8 f8_operand(PyObject *pair, const char *name)
{
    PyObject *d = nullptr, *s = nullptr;
    if (PyTuple_Check(pair) && PyTuple_GET_SIZE(pair) == 2) {
        d = PyTuple_GET_ITEM(pair, 0);
        s = PyTuple_GET_ITEM(pair, 1);
    } else if (PyList_Check(pair) && PyList_GET_SIZE(pair) == 2) {
        d = PyList_GET_ITEM(pair, 0);
        s = PyList_GET_ITEM(pair, 1);
    } else {
        fail(PyExc_TypeError, std::string("f8_matmul: ") + name + " must be (data, scale)");
    }
    const at::Tensor &data = need(d), &scale = need(s);
    on_gpu(data);
    beside(scale, data, "f8_matmul");
    F8 m;
    m.fmt = f8_code(data.scalar_type());
    if (m.fmt < 0 || data.dim() != 2 || scale.dim() != 2 ||
        (scale.scalar_type() != at::kFloat8_e8m0fnu && scale.scalar_type() != at::kByte))
        fail(PyExc_TypeError, std::string("f8_matmul: ") + name + " must be a float8 matrix and its E8M0 scales");
    m.R = data.size(0);
    m.C = data.size(1);
    const long long nb = (m.C + 127) / 128, blocks = (m.R + 127) / 128;
    if (scale.size(1) != nb || (scale.size(0) != m.R && scale.size(0) != blocks))
        fail(PyExc_ValueError, std::string("f8_matmul: ") + name + " " + shape(data) + " needs scales [" +
                                   std::to_string(m.R) + " or " + std::to_string(blocks) + ", " + std::to_string(nb) +
                                   "], got " + shape(scale));
    m.square = scale.size(0) != m.R;
    m.data = bordered(data, 16, m.ld);
    m.scale = bordered(scale, 4, m.lds);
    return m;
}

// x [R, C] -> rows form, columns form, column sums [ceil(R / 128), C] (each where asked for)
struct Quant {
    F8 rows, cols;
    at::Tensor sums;
};
Quant f8_quant(const at::Tensor &x, int fmt, bool square, bool rows, bool cols, bool sums, void *st)
{
    on_gpu(x);
    if (x.dim() != 2) fail(PyExc_ValueError, "8-bit rows are made from a matrix, got " + shape(x));
    const int code = type_code(x.scalar_type());
    if (code < 0) fail(PyExc_TypeError, "8-bit rows are made from float32, bfloat16 or float16");
    if (fmt != LCF_E4M3 && fmt != LCF_E5M2) fail(PyExc_TypeError, "8-bit rows are float8_e4m3fn or float8_e5m2");
    const int R = count(x.size(0), "8-bit rows"), C = count(x.size(1), "8-bit rows");
    const Rows v = rows_of(x, C);
    Quant q;
    if (rows) q.rows = f8_empty(R, C, square, fmt, x);
    if (cols) q.cols = f8_empty(C, R, square, fmt, x);
    if (sums) q.sums = at::empty({(R + 127) / 128, C}, x.options().dtype(at::kFloat));
    if (R && C)
        check(L.f8_quant(v.ptr(), v.ld, R, C, code, fmt, square, rows ? q.rows.q() : nullptr, q.rows.ld,
                         rows ? q.rows.s() : nullptr, (int)q.rows.lds, cols ? q.cols.q() : nullptr, q.cols.ld,
                         cols ? q.cols.s() : nullptr, (int)q.cols.lds, sums ? (float *)q.sums.data_ptr() : nullptr,
                         st));
    return q;
}

void check_affine(const at::Tensor *v, long long N, const at::Tensor &like, const char *name)
{
    if (!v) return;
    beside(*v, like, "f8_matmul");
    if (v->scalar_type() != at::kFloat || v->dim() != 1 || v->size(0) != N || !v->is_contiguous())
        fail(PyExc_ValueError, std::string("f8_matmul: ") + name + " must be " + std::to_string(N) + " contiguous float32");
}
float *ptr(const at::Tensor *t) { return t ? (float *)t->data_ptr() : nullptr; }

at::Tensor f8_mm(const F8 &a, const F8 &b, const at::Tensor *scale, const at::Tensor *shift, bool relu, int code,
                 const at::Tensor *to, void *st)
{
    if (a.C != b.C)
        fail(PyExc_ValueError, "f8_matmul: " + shape(a.data) + " against " + shape(b.data) + ": the last dimensions must agree");
    if (a.square) fail(PyExc_ValueError, "f8_matmul: a needs one scale for each row and 128 columns");
    beside(b.data, a.data, "f8_matmul");
    const int M = count(a.R, "f8_matmul"), N = count(b.R, "f8_matmul"), K = count(a.C, "f8_matmul");
    check_affine(scale, N, a.data, "scale");
    check_affine(shift, N, a.data, "shift");
    at::Tensor out;
    if (to) {
        out = *to;
        code = type_code(out.scalar_type());
        if (!out.is_cuda() || out.get_device() != a.data.get_device() || code < 0 || out.dim() != 2 ||
            out.size(0) != M || out.size(1) != N || (N > 1 && out.stride(1) != 1) || (M > 1 && out.stride(0) < N))
            fail(PyExc_ValueError, "f8_matmul: out must be a float matrix [" + std::to_string(M) + ", " +
                                       std::to_string(N) + "] with unit stride in a row on the operands' device");
    } else {
        if (code < 0) fail(PyExc_TypeError, "f8_matmul: out_dtype must be float32, bfloat16 or float16");
        out = at::empty({M, N}, a.data.options().dtype(type_of(code)));
    }
    const size_t n = L.f8_gemm_workspace_bytes(M, N, K, code);
    at::Tensor ws;
    if (n) ws = bytes(n, a.data);
    check(L.f8_gemm(K ? a.q() : nullptr, a.ld, K ? a.s() : nullptr, (int)a.lds, a.fmt, K ? b.q() : nullptr, b.ld,
                    K ? b.s() : nullptr, (int)b.lds, b.fmt, b.square, M, N, K, ptr(scale), ptr(shift), relu,
                    out.data_ptr(), M > 1 ? (long long)out.stride(0) : N, code, n ? ws.data_ptr() : nullptr,
                    n ? (size_t)ws.numel() : 0, st));
    return out;
}

// x's rows through b in one launch, of x's own type; undefined where lcf_f8_linear does not take the sizes
at::Tensor f8_fused(const at::Tensor &x, const F8 &b, const at::Tensor *scale, const at::Tensor *shift, bool relu, void *st)
{
    on_gpu(x);
    const int code = type_code(x.scalar_type());
    if (code < 0 || x.dim() != 2 || x.size(1) != b.C)
        fail(PyExc_ValueError, "f8_linear: rows " + shape(x) + " against " + shape(b.data));
    beside(b.data, x, "f8_linear");
    const int M = count(x.size(0), "f8_linear"), N = count(b.R, "f8_linear"), K = count(b.C, "f8_linear");
    if (M < 4096 || N > 256 || K > 512 || b.fmt != LCF_E4M3) return at::Tensor(); // far from thin: nothing to ask
    check_affine(scale, N, x, "scale");
    check_affine(shift, N, x, "shift");
    const Rows v = rows_of(x, K);
    at::Tensor out = at::empty({M, N}, x.options());
    const int rc = L.f8_linear(v.ptr(), v.ld, code, b.q(), b.ld, b.s(), (int)b.lds, b.square, M, N, K, ptr(scale),
                               ptr(shift), relu, out.data_ptr(), N, code, st);
    if (rc == LCF_ERR_UNSUPPORTED) return at::Tensor();
    check(rc);
    return out;
}
at::Tensor f8_product(const at::Tensor &x, const F8 &b, const at::Tensor *scale, const at::Tensor *shift, bool relu,
                      void *st)
{
    const at::Tensor out = f8_fused(x, b, scale, shift, relu, st);
    if (out.defined()) return out;
    return f8_mm(f8_quant(x, LCF_E4M3, false, true, false, false, st).rows, b, scale, shift, relu,
                 type_code(x.scalar_type()), nullptr, st);
}

F8 weight_image(const at::Tensor &w, bool transpose, int fmt, void *st)
{
    Quant q = f8_quant(w, fmt, true, !transpose, transpose, false, st);
    return transpose ? q.cols : q.rows;
}

// ---- entry points
using Args = PyObject *const *;
template <typename F> PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F f)
{
    try {
        if (got != want) fail(PyExc_TypeError, "wrong number of arguments");
        if (!L.strerror) fail(PyExc_RuntimeError, "row_ops: bind() first");
        at::AutoDispatchBelowADInplaceOrView below; // nothing here is recorded by autograd
        return f();
    } catch (const Err &e) {
        PyErr_SetString(e.type, e.what.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "row_ops: unknown error");
    }
    return nullptr;
}

PyObject *py_bind(PyObject *, Args a, Py_ssize_t n)
{
    if (n != 1 || !PyDict_Check(a[0])) {
        PyErr_SetString(PyExc_TypeError, "bind(addresses)");
        return nullptr;
    }
    Lib l{};
#define F(name)                                                                                     \
    {                                                                                               \
        PyObject *p = PyDict_GetItemString(a[0], "lcf_" #name);                                     \
        if (!p) {                                                                                   \
            PyErr_SetString(PyExc_KeyError, "lcf_" #name);                                          \
            return nullptr;                                                                         \
        }                                                                                           \
        l.name = (decltype(l.name))PyLong_AsVoidPtr(p);                                             \
    }
    LCF_FUNCTIONS(F)
#undef F
    L = l;
    Py_RETURN_NONE;
}

// f8_quant(x, format, square, rows, cols, stream) -> (data, scale, data^T, scale^T)
PyObject *py_f8_quant(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 6, [&] {
        const Quant q = f8_quant(need(a[0]), (int)number(a[1]), truth(a[2]), truth(a[3]), truth(a[4]), false, stream_of(a[5]));
        return tuple(q.rows.data, q.rows.scale, q.cols.data, q.cols.scale);
    });
}
// f8_rows(x, format, stream) -> (data, scale)
PyObject *py_f8_rows(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 3, [&] {
        const Quant q = f8_quant(need(a[0]), (int)number(a[1]), false, true, false, false, stream_of(a[2]));
        return tuple(q.rows.data, q.rows.scale);
    });
}
// f8_mm(a, b, scale, shift, relu, out type, out, stream)
PyObject *py_f8_mm(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 8, [&] {
        return wrap(f8_mm(f8_operand(a[0], "a"), f8_operand(a[1], "b"), maybe(a[2]), maybe(a[3]), truth(a[4]),
                          (int)number(a[5]), maybe(a[6]), stream_of(a[7])));
    });
}
// f8_product(x, b, scale, shift, relu, stream)
PyObject *py_f8_product(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 6, [&] {
        return wrap(f8_product(need(a[0]), f8_operand(a[1], "b"), maybe(a[2]), maybe(a[3]), truth(a[4]), stream_of(a[5])));
    });
}
// f8_linear_fwd(x, weight, bias, turned, x8, stream) -> y
PyObject *py_f8_linear_fwd(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 6, [&] {
        const at::Tensor &x = need(a[0]), &w = need(a[1]);
        on_gpu(x);
        beside(w, x, "f8_linear");
        void *st = stream_of(a[5]);
        const F8 image = weight_image(w, truth(a[3]), LCF_E4M3, st);
        at::Tensor shift;
        if (const at::Tensor *b = maybe(a[2])) {
            beside(*b, x, "f8_linear");
            shift = b->to(at::kFloat).contiguous();
        }
        const at::Tensor *sh = shift.defined() ? &shift : nullptr;
        if (a[4] == Py_None) return wrap(f8_product(x, image, nullptr, sh, false, st));
        return wrap(f8_mm(f8_operand(a[4], "x8"), image, nullptr, sh, false, type_code(x.scalar_type()), nullptr, st));
    });
}
// f8_linear_bwd(dy, x, weight, turned, need dx, need dw, bias type or None, stream) -> (dx, dw, db)
PyObject *py_f8_linear_bwd(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 8, [&] {
        const at::Tensor &x = need(a[1]), &w = need(a[2]);
        const bool turned = truth(a[3]), need_x = truth(a[4]), need_w = truth(a[5]), need_b = a[6] != Py_None;
        void *st = stream_of(a[7]);
        at::Tensor dy = need(a[0]);
        beside(dy, x, "f8_linear");
        if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
        at::Tensor dx, dw, db;
        // the input's gradient takes dy as it is where one launch does both; elsewhere dy's rows form, its
        // columns form and the bias's sums come out of one reading
        F8 image;
        if (need_x) {
            image = weight_image(w, !turned, LCF_E4M3, st);
            dx = f8_fused(dy, image, nullptr, nullptr, false, st);
        }
        const bool rows = need_x && !dx.defined();
        Quant q;
        if (rows || need_w || need_b) q = f8_quant(dy, LCF_E4M3, false, rows, need_w, need_b, st);
        if (rows) dx = f8_mm(q.rows, image, nullptr, nullptr, false, type_code(dy.scalar_type()), nullptr, st);
        if (need_w) {
            const F8 xt = f8_quant(x, LCF_E4M3, false, false, true, false, st).cols;
            dw = f8_mm(turned ? xt : q.cols, turned ? q.cols : xt, nullptr, nullptr, false, type_code(w.scalar_type()),
                       nullptr, st);
        }
        if (need_b) {
            const int code = (int)number(a[6]);
            const int C = (int)dy.size(1);
            db = at::empty({C}, dy.options().dtype(type_of(code)));
            if (C) check(L.sum_parts((const float *)q.sums.data_ptr(), (int)q.sums.size(0), C, db.data_ptr(), code, st));
        }
        return tuple(dx, dw, db);
    });
}

// rms_fwd(x, weight, eps, residual, want y, want inv, 8-bit format or -1, stream)
//   -> (y, h, inv, data, scale); h is None without a residual
PyObject *py_rms_fwd(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 8, [&] {
        const at::Tensor &x = need(a[0]);
        const at::Tensor *w = maybe(a[1]), *r = maybe(a[3]);
        const double eps = real(a[2]);
        const int fmt = (int)number(a[6]), code = type_code(x.scalar_type());
        on_gpu(x);
        if (code < 0 || x.dim() < 1) fail(PyExc_TypeError, "rms_norm: rows must be float32, bfloat16 or float16");
        const long long width = x.size(-1);
        if (width < 1 || width > 16384)
            fail(PyExc_ValueError, "rms_norm: 1 to 16384 columns, got " + std::to_string(width));
        if (!(eps >= 0.0)) fail(PyExc_ValueError, "rms_norm: eps must not be negative");
        at::Tensor wc;
        if (w) {
            beside(*w, x, "rms_norm");
            if (type_code(w->scalar_type()) < 0 || w->dim() != 1 || w->size(0) != width)
                fail(PyExc_ValueError, "rms_norm: weight must be a float tensor of " + std::to_string(width) + " elements");
            wc = w->contiguous();
        }
        if (r) {
            beside(*r, x, "rms_norm");
            if (r->sizes() != x.sizes() || r->scalar_type() != x.scalar_type())
                fail(PyExc_ValueError, "rms_norm: residual must have x's shape and type");
        }
        if (fmt >= 0 && x.dim() != 2) fail(PyExc_ValueError, "rms_norm_f8: x must be [rows, columns]");
        const Rows v = rows_of(x, width), rv = r ? rows_of(*r, width) : Rows{at::Tensor(), 0, 0};
        const int rows = count(v.n, "rms_norm");
        at::Tensor y, h, inv;
        if (truth(a[4])) y = at::empty(x.sizes(), x.options());
        if (r) h = at::empty(x.sizes(), x.options());
        if (truth(a[5])) inv = at::empty({rows}, x.options().dtype(at::kFloat));
        F8 q;
        if (fmt >= 0) q = f8_empty(rows, width, false, fmt, x);
        check(L.rms_norm_fwd(v.ptr(), v.ld, r ? rv.ptr() : nullptr, rv.ld, rows, (int)width, code,
                             w ? wc.data_ptr() : nullptr, w ? type_code(wc.scalar_type()) : 0, (float)eps,
                             y.defined() ? y.data_ptr() : nullptr, r ? h.data_ptr() : nullptr,
                             inv.defined() ? (float *)inv.data_ptr() : nullptr, fmt >= 0 && rows ? q.q() : nullptr, q.ld,
                             fmt >= 0 && rows ? q.s() : nullptr, (int)q.lds, fmt >= 0 ? fmt : 0, stream_of(a[7])));
        return tuple(y, h, inv, q.data, q.scale);
    });
}
// rms_bwd(h, weight, inv, dy, dh, need dw, stream) -> (dx, dw)
PyObject *py_rms_bwd(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 7, [&] {
        const at::Tensor &h = need(a[0]), &inv = need(a[2]);
        const at::Tensor *w = maybe(a[1]), *g = maybe(a[4]);
        at::Tensor dy = need(a[3]), dh;
        const long long width = h.size(-1);
        const int code = type_code(h.scalar_type());
        beside(dy, h, "rms_norm");
        if (dy.sizes() != h.sizes()) fail(PyExc_ValueError, "rms_norm: a gradient of another shape");
        if (dy.scalar_type() != h.scalar_type()) dy = dy.to(h.scalar_type());
        if (g) {
            beside(*g, h, "rms_norm");
            if (g->sizes() != h.sizes()) fail(PyExc_ValueError, "rms_norm: a gradient of another shape");
            dh = g->scalar_type() == h.scalar_type() ? *g : g->to(h.scalar_type());
        }
        const Rows hv = rows_of(h, width), dv = rows_of(dy, width), gv = g ? rows_of(dh, width) : Rows{at::Tensor(), 0, 0};
        const int rows = count(hv.n, "rms_norm");
        at::Tensor dx = at::empty(h.sizes(), h.options()), dw, ws, wc;
        if (w) wc = w->contiguous();
        if (w && truth(a[5])) {
            dw = at::empty({width}, w->options());
            ws = bytes(L.rms_norm_workspace_bytes(rows, (int)width), h);
        }
        check(L.rms_norm_bwd(hv.ptr(), hv.ld, dv.ptr(), dv.ld, g ? gv.ptr() : nullptr, gv.ld, rows, (int)width, code,
                             w ? wc.data_ptr() : nullptr, w ? type_code(wc.scalar_type()) : 0, (const float *)inv.data_ptr(),
                             dx.data_ptr(), dw.defined() ? dw.data_ptr() : nullptr, ws.defined() ? ws.data_ptr() : nullptr,
                             ws.defined() ? (size_t)ws.numel() : 0, stream_of(a[6])));
        return tuple(dx, dw);
    });
}

// clip(tensors, out or None, p, max_norm or None, stream) -> norm.  max_norm None: the norm alone.
PyObject *py_clip(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 5, [&] {
        if (!PyList_Check(a[0])) fail(PyExc_TypeError, "expected a list of tensors");
        const Py_ssize_t k = PyList_GET_SIZE(a[0]);
        if (k == 0) fail(PyExc_ValueError, "expected at least one tensor");
        const bool clip = a[3] != Py_None, list = clip && PyList_Check(a[1]), flat = clip && !list && a[1] != Py_None;
        if (list && PyList_GET_SIZE(a[1]) != k) fail(PyExc_ValueError, "out must have a tensor for each gradient");
        std::vector<lcf_grad> t((size_t)k);
        const at::Tensor &first = need(PyList_GET_ITEM(a[0], 0));
        on_gpu(first);
        long long total = 0;
        auto take = [&](PyObject *o, const char *what) -> const at::Tensor & {
            const at::Tensor &g = need(o);
            on_gpu(g);
            if (g.get_device() != first.get_device())
                fail(PyExc_RuntimeError, "the tensors of one norm must be on one device");
            if (type_code(g.scalar_type()) < 0)
                fail(PyExc_TypeError, std::string(what) + " must be float32, bfloat16 or float16");
            if (!g.is_non_overlapping_and_dense())
                fail(PyExc_ValueError, std::string(what) + " must be dense in memory (got a strided view " + shape(g) +
                                           "): pass .contiguous()");
            return g;
        };
        for (Py_ssize_t i = 0; i < k; ++i) {
            const at::Tensor &g = take(PyList_GET_ITEM(a[0], i), "gradients");
            lcf_grad &e = t[(size_t)i];
            e.g = g.data_ptr();
            e.n = g.numel();
            e.dtype = e.out_dtype = type_code(g.scalar_type());
            e.out = const_cast<void *>(e.g);
            total += e.n;
            if (list) {
                const at::Tensor &o = take(PyList_GET_ITEM(a[1], i), "out");
                // the same order in memory: sizes and, where they say something, strides
                if (o.sizes() != g.sizes() || (o.numel() > 1 && o.strides() != g.strides()))
                    fail(PyExc_ValueError, "out must be tensors of the gradients' sizes and strides");
                e.out = o.data_ptr();
                e.out_dtype = type_code(o.scalar_type());
            }
        }
        if (flat) {
            const at::Tensor &o = take(a[1], "out");
            if (!o.is_contiguous() || o.numel() != total)
                fail(PyExc_ValueError, "out must be a contiguous tensor with as many elements as the gradients have together");
            char *at = (char *)o.data_ptr();
            for (lcf_grad &e : t) {
                e.out = at;
                e.out_dtype = type_code(o.scalar_type());
                at += e.n * o.element_size();
            }
        }
        at::Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
        at::Tensor ws = bytes(L.grad_norm_workspace_bytes((int)k), first);
        if (clip)
            check(L.grad_clip(t.data(), (int)k, (int)number(a[2]), (float)real(a[3]), (float *)norm.data_ptr(),
                              ws.data_ptr(), (size_t)ws.numel(), stream_of(a[4])));
        else
            check(L.grad_norm(t.data(), (int)k, (int)number(a[2]), (float *)norm.data_ptr(), ws.data_ptr(),
                              (size_t)ws.numel(), stream_of(a[4])));
        return wrap(norm);
    });
}

#define METHOD(name) {#name, (PyCFunction)(void (*)())py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),          METHOD(f8_quant),      METHOD(f8_rows), METHOD(f8_mm),   METHOD(f8_product),
                         METHOD(f8_linear_fwd), METHOD(f8_linear_bwd), METHOD(rms_fwd), METHOD(rms_bwd), METHOD(clip),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_row_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__row_ops(void) { return PyModule_Create(&module); }
