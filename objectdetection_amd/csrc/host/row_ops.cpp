// row_ops.cpp -- the host side of the row operators (grad_norm.hip, rms_norm.hip, f8.hip): argument
// checks, output allocation and the calls into liblcf's C ABI, as a CPython module over torch's C++
// tensors.  These operators are called on one row as often as on many, and then the host's time is
// all there is: the same checks in Python took 15 to 40 us a call, and 80 us for a list of 78
// gradients.  The library's functions are handed over by address (objectdetection_amd/_lib.py loads
// it), so there is one liblcf in a process and nothing is linked against.
// Work goes to the current stream of the tensors' device, which is made the current one meanwhile.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../../include/lcf.h"

namespace {

// a refusal, with the Python exception it becomes (a std::exception: autograd's threads take no other)
struct Err : std::runtime_error {
    PyObject *type;
    Err(PyObject *t, const std::string &what) : std::runtime_error(what), type(t) {}
};
[[noreturn]] void fail(PyObject *type, const std::string &what) { throw Err(type, what); }

#define LCF_FUNCTIONS(F)                                                                                       \
    F(strerror) F(grad_norm_workspace_bytes) F(grad_norm) F(grad_clip) F(rms_norm_fwd) F(rms_norm_workspace_bytes) \
    F(rms_norm_bwd) F(f8_quant) F(f8_gemm_split_bytes) F(f8_gemm) F(f8_linear) F(sum_parts) \
    F(f8_weight_grad_workspace_bytes) F(f8_weight_grad)
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
// the device of x made current for a scope, and its current stream
struct On {
    c10::DeviceGuard guard;
    void *st;
    explicit On(const at::Tensor &x) : guard((on_gpu(x), x.device())), st(c10::hip::getCurrentHIPStream(x.get_device()).stream()) {}
};
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
// a kernel is about to write t: what has saved it for a backward pass, or keeps a form of it, can tell
void written(const at::Tensor &t) { t.unsafeGetTensorImpl()->bump_version(); }
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

F8 f8_operand(const at::Tensor &data, const at::Tensor &scale, const char *name)
{
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
    return f8_operand(need(d), need(s), name);
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
    const size_t n = L.f8_gemm_split_bytes(M, N, K, code);
    at::Tensor ws;
    if (n) ws = bytes(n, a.data);
    if (to) written(out);
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

// ---- entry points
using Args = PyObject *const *;
template <typename F> PyObject *guarded_grad(Py_ssize_t got, Py_ssize_t want, F f)
{
    try {
        if (got != want) fail(PyExc_TypeError, "wrong number of arguments");
        if (!L.strerror) fail(PyExc_RuntimeError, "row_ops: bind() first");
        return f();
    } catch (const Err &e) {
        PyErr_SetString(e.type, e.what());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "row_ops: unknown error");
    }
    return nullptr;
}

template <typename F> PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F f)
{
    return guarded_grad(got, want, [&] {
        at::AutoDispatchBelowADInplaceOrView below; // nothing in here is recorded by autograd
        return f();
    });
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

// ---- the operators with their gradients
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;
const Tensor *maybe(const Maybe &t) { return t && t->defined() ? &*t : nullptr; }
// the gradients are kernels' outputs, with no graph of their own: one made for a second derivative
// (create_graph) would leave their share out without a word
void once(const char *who)
{
    if (at::GradMode::is_enabled())
        fail(PyExc_RuntimeError, std::string(who) + " is differentiable once: no backward pass with create_graph=True");
}
bool wants(const Tensor *t) { return t && t->requires_grad(); }
// a forward-mode tangent needs no requires_grad: the unrecorded path would drop it without a word
void no_tangent(const char *who, std::initializer_list<const Tensor *> inputs)
{
    for (const Tensor *t : inputs)
        if (t && t->_fw_grad(0).defined())
            fail(PyExc_RuntimeError, std::string(who) + " has no forward-mode derivative");
}

struct Normed {
    Tensor y, h, inv;
    F8 q;
};
Normed rms_fwd(const Tensor &x, const Tensor *w, double eps, const Tensor *r, bool want_y, bool want_inv, int fmt)
{
    const On on(x);
    const int code = type_code(x.scalar_type());
    if (code < 0 || x.dim() < 1) fail(PyExc_TypeError, "rms_norm: rows must be float32, bfloat16 or float16");
    const long long width = x.size(-1);
    if (width < 1 || width > 16384) fail(PyExc_ValueError, "rms_norm: 1 to 16384 columns, got " + std::to_string(width));
    if (!(eps >= 0.0)) fail(PyExc_ValueError, "rms_norm: eps must not be negative");
    Tensor wc;
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
    const Rows v = rows_of(x, width), rv = r ? rows_of(*r, width) : Rows{Tensor(), 0, 0};
    const int rows = count(v.n, "rms_norm");
    Normed o;
    if (want_y) o.y = at::empty(x.sizes(), x.options());
    if (r) o.h = at::empty(x.sizes(), x.options());
    if (want_inv) o.inv = at::empty({rows}, x.options().dtype(at::kFloat));
    const bool q8 = fmt >= 0;
    if (q8) o.q = f8_empty(rows, width, false, fmt, x);
    check(L.rms_norm_fwd(v.ptr(), v.ld, r ? rv.ptr() : nullptr, rv.ld, rows, (int)width, code, w ? wc.data_ptr() : nullptr,
                         w ? type_code(wc.scalar_type()) : 0, (float)eps, want_y ? o.y.data_ptr() : nullptr,
                         r ? o.h.data_ptr() : nullptr, want_inv ? (float *)o.inv.data_ptr() : nullptr,
                         q8 && rows ? o.q.q() : nullptr, o.q.ld, q8 && rows ? o.q.s() : nullptr, (int)o.q.lds, q8 ? fmt : 0,
                         on.st));
    return o;
}

// y (and h = x + residual) from x; backward from h and the rows' inverse root mean squares.  x and the
// residual share one gradient.
struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &w, double eps, const Maybe &r)
    {
        const Normed o = rms_fwd(x, maybe(w), eps, maybe(r), true, true, -1);
        ctx->saved_data["two"] = maybe(r) != nullptr;
        ctx->save_for_backward({maybe(r) ? o.h : x, w ? *w : Tensor(), o.inv});
        ctx->set_materialize_grads(false);
        if (maybe(r)) return {o.y, o.h};
        return {o.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once("rms_norm");
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list saved = ctx->get_saved_variables();
        const bool two = ctx->saved_data["two"].toBool();
        const Tensor &h = saved[0], &w = saved[1];
        const bool need_w = w.defined() && ctx->needs_input_grad(1);
        Tensor dy = grads[0], dh = two ? grads[1] : Tensor();
        if (!dy.defined()) { // the norm's output was not used: the sum's gradient passes through
            return {dh, need_w && dh.defined() ? at::zeros_like(w) : Tensor(), Tensor(), two ? dh : Tensor()};
        }
        const On on(h);
        const long long width = h.size(-1);
        if (dy.scalar_type() != h.scalar_type()) dy = dy.to(h.scalar_type());
        if (dh.defined() && dh.scalar_type() != h.scalar_type()) dh = dh.to(h.scalar_type());
        const Rows hv = rows_of(h, width), dv = rows_of(dy, width),
                   gv = dh.defined() ? rows_of(dh, width) : Rows{Tensor(), 0, 0};
        const int rows = count(hv.n, "rms_norm"), code = type_code(h.scalar_type());
        Tensor dx = at::empty(h.sizes(), h.options()), dw, ws, wc;
        if (w.defined()) wc = w.contiguous();
        if (need_w) {
            dw = at::empty({width}, w.options());
            ws = bytes(L.rms_norm_workspace_bytes(rows, (int)width), h);
        }
        check(L.rms_norm_bwd(hv.ptr(), hv.ld, dv.ptr(), dv.ld, dh.defined() ? gv.ptr() : nullptr, gv.ld, rows, (int)width,
                             code, w.defined() ? wc.data_ptr() : nullptr, w.defined() ? type_code(wc.scalar_type()) : 0,
                             (const float *)saved[2].data_ptr(), dx.data_ptr(), need_w ? dw.data_ptr() : nullptr,
                             need_w ? ws.data_ptr() : nullptr, need_w ? (size_t)ws.numel() : 0, on.st));
        return {dx, dw, Tensor(), two ? dx : Tensor()};
    }
};

// back: the image that the input's gradient takes, made from the same reading of the weight
Tensor f8_linear_fwd(const Tensor &x, const Tensor &w, const Tensor *bias, bool turned, const F8 *x8, F8 *back)
{
    const On on(x);
    beside(w, x, "f8_linear");
    const Quant q = f8_quant(w, LCF_E4M3, true, !turned || back, turned || back, false, on.st);
    const F8 &image = turned ? q.cols : q.rows;
    if (back) *back = turned ? q.rows : q.cols;
    Tensor shift;
    if (bias) {
        beside(*bias, x, "f8_linear");
        shift = bias->to(at::kFloat).contiguous();
    }
    const Tensor *sh = bias ? &shift : nullptr;
    if (!x8) return f8_product(x, image, nullptr, sh, false, on.st);
    return f8_mm(*x8, image, nullptr, sh, false, type_code(x.scalar_type()), nullptr, on.st);
}

// dw of type code w and, with bias >= 0, db of that type, where lcf_f8_weight_grad takes the sizes; false elsewhere
bool f8_weight_grad(const Tensor &x, const Tensor &dy, bool turned, int w, int bias, Tensor &dw, Tensor &db, void *st)
{
    const int R = count(x.size(0), "f8_linear"), K = count(x.size(1), "f8_linear"), N = count(dy.size(1), "f8_linear");
    const size_t n = L.f8_weight_grad_workspace_bytes(R, K, N);
    if (!n) return false;
    const Rows xv = rows_of(x, K), dv = rows_of(dy, N);
    const Tensor ws = bytes(n, x), to = at::empty({turned ? K : N, turned ? N : K}, x.options().dtype(type_of(w))),
                 sum = bias >= 0 ? at::empty({N}, x.options().dtype(type_of(bias))) : Tensor();
    const int rc = L.f8_weight_grad(xv.ptr(), xv.ld, dv.ptr(), dv.ld, R, K, N, type_code(x.scalar_type()), turned,
                                    to.data_ptr(), w, bias >= 0 ? sum.data_ptr() : nullptr,
                                    bias >= 0 ? bias : 0, ws.data_ptr(), (size_t)ws.numel(), st);
    if (rc == LCF_ERR_UNSUPPORTED) return false;
    check(rc);
    dw = to;
    db = sum;
    return true;
}

// y = x W^T (+ bias) with x and W rounded to 8-bit form.  The three products (y, dx = dy W, dW = dy^T x)
// run on 8-bit operands, each operand's scale blocks lying along the axis that its product sums over;
// the rounding is passed through unchanged.  turned: the weight is stored [K, N].
struct F8Linear : torch::autograd::Function<F8Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Maybe &bias, bool turned,
                          const F8 *x8)
    {
        F8 back;
        Tensor y = f8_linear_fwd(x, w, maybe(bias), turned, x8, x.requires_grad() ? &back : nullptr);
        // the rows are for the weight's gradient alone, and of the weight its type is enough: what is not kept
        // costs no memory and may be written to
        ctx->save_for_backward({w.requires_grad() ? x : Tensor(), back.data, back.scale});
        ctx->saved_data["turned"] = turned;
        ctx->saved_data["x"] = (int64_t)type_code(x.scalar_type());
        ctx->saved_data["w"] = (int64_t)type_code(w.scalar_type());
        ctx->saved_data["bias"] = (int64_t)(maybe(bias) ? type_code(bias->scalar_type()) : -1);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once("f8_linear");
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0];
        const bool turned = ctx->saved_data["turned"].toBool();
        const int w = (int)ctx->saved_data["w"].toInt(), bias = (int)ctx->saved_data["bias"].toInt();
        const bool need_x = ctx->needs_input_grad(0);
        bool need_w = ctx->needs_input_grad(1), need_b = bias >= 0 && ctx->needs_input_grad(2);
        Tensor dy = grads[0], dx, dw, db;
        const On on(dy);
        const at::ScalarType rows_type = type_of((int)ctx->saved_data["x"].toInt());
        if (dy.scalar_type() != rows_type) dy = dy.to(rows_type);
        // the input's gradient takes dy as it is where one launch does both; elsewhere dy's rows form, its
        // columns form and the bias's sums come out of one reading
        F8 image;
        if (need_x) {
            image = f8_operand(saved[1], saved[2], "weight");
            dx = f8_fused(dy, image, nullptr, nullptr, false, on.st);
        }
        // the weight's gradient and the bias's take both as they are where one kernel does all
        bool done = false;
        if (need_w) done = f8_weight_grad(x, dy, turned, w, need_b ? bias : -1, dw, db, on.st);
        const bool rows = need_x && !dx.defined();
        need_w = need_w && !done;
        need_b = need_b && !done;
        Quant q;
        if (rows || need_w || need_b) q = f8_quant(dy, LCF_E4M3, false, rows, need_w, need_b, on.st);
        if (rows) dx = f8_mm(q.rows, image, nullptr, nullptr, false, type_code(dy.scalar_type()), nullptr, on.st);
        if (need_w) {
            const F8 xt = f8_quant(x, LCF_E4M3, false, false, true, false, on.st).cols;
            dw = f8_mm(turned ? xt : q.cols, turned ? q.cols : xt, nullptr, nullptr, false, w, nullptr, on.st);
        }
        if (need_b) {
            const int C = (int)dy.size(1);
            db = at::empty({C}, dy.options().dtype(type_of(bias)));
            if (C) check(L.sum_parts((const float *)q.sums.data_ptr(), (int)q.sums.size(0), C, db.data_ptr(), bias, on.st));
        }
        return {dx, dw, db, Tensor(), Tensor()};
    }
};

// f8_quant(x, format, square, rows, cols) -> (data, scale, data^T, scale^T)
PyObject *py_f8_quant(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 5, [&] {
        const Tensor &x = need(a[0]);
        const On on(x);
        const Quant q = f8_quant(x, (int)number(a[1]), truth(a[2]), truth(a[3]), truth(a[4]), false, on.st);
        return tuple(q.rows.data, q.rows.scale, q.cols.data, q.cols.scale);
    });
}
// f8_rows(x, format) -> (data, scale)
PyObject *py_f8_rows(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 2, [&] {
        const Tensor &x = need(a[0]);
        const On on(x);
        const Quant q = f8_quant(x, (int)number(a[1]), false, true, false, false, on.st);
        return tuple(q.rows.data, q.rows.scale);
    });
}
// f8_mm(a, b, scale, shift, relu, out type, out)
PyObject *py_f8_mm(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 7, [&] {
        const F8 x = f8_operand(a[0], "a"), b = f8_operand(a[1], "b");
        const On on(x.data);
        return wrap(f8_mm(x, b, maybe(a[2]), maybe(a[3]), truth(a[4]), (int)number(a[5]), maybe(a[6]), on.st));
    });
}
// f8_product(x, b, scale, shift, relu)
PyObject *py_f8_product(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 5, [&] {
        const Tensor &x = need(a[0]);
        const On on(x);
        return wrap(f8_product(x, f8_operand(a[1], "b"), maybe(a[2]), maybe(a[3]), truth(a[4]), on.st));
    });
}
// f8_linear(x, weight, bias, turned, x8) -> y, differentiable
PyObject *py_f8_linear(PyObject *, Args a, Py_ssize_t n)
{
    return guarded_grad(n, 5, [&] {
        const Tensor &x = need(a[0]), &w = need(a[1]);
        const Tensor *bias = maybe(a[2]);
        const bool turned = truth(a[3]);
        no_tangent("f8_linear", {&x, &w, bias});
        on_gpu(x);
        if (type_code(x.scalar_type()) < 0 || type_code(w.scalar_type()) < 0 || x.dim() != 2 || w.dim() != 2 ||
            x.size(1) != w.size(turned ? 0 : 1))
            fail(PyExc_ValueError, "f8_linear: x " + shape(x) + " against weight " + shape(w) +
                                       " (float32, bfloat16 or float16)");
        if (at::GradMode::is_enabled() && (wants(&w) || wants(bias)) && x.size(0) > 1 << 22)
            fail(PyExc_ValueError, "f8_linear: at most 2^22 rows where weight or bias wants a gradient (a sum over them)");
        const long long out = w.size(turned ? 1 : 0);
        if (x.size(1) > 1 << 22 || out > 1 << 22) fail(PyExc_ValueError, "f8_linear: at most 2^22 columns");
        if (bias && (bias->dim() != 1 || bias->size(0) != out || type_code(bias->scalar_type()) < 0))
            fail(PyExc_ValueError, "f8_linear: bias must have " + std::to_string(out) + " float elements");
        F8 x8;
        if (a[4] != Py_None) {
            x8 = f8_operand(a[4], "x8");
            if (x8.R != x.size(0) || x8.C != x.size(1)) fail(PyExc_ValueError, "f8_linear: x8 must be the 8-bit form of x");
        }
        const F8 *p8 = a[4] != Py_None ? &x8 : nullptr;
        if (at::GradMode::is_enabled() && (wants(&x) || wants(&w) || wants(bias)))
            return wrap(F8Linear::apply(x, w, bias ? Maybe(*bias) : Maybe(), turned, p8));
        at::AutoDispatchBelowADInplaceOrView below;
        return wrap(f8_linear_fwd(x, w, bias, turned, p8, nullptr));
    });
}
// rms_norm(x, weight, eps, residual) -> y, or (y, h) with a residual; differentiable
PyObject *py_rms_norm(PyObject *, Args a, Py_ssize_t n)
{
    return guarded_grad(n, 4, [&]() -> PyObject * {
        const Tensor &x = need(a[0]);
        const Tensor *w = maybe(a[1]), *r = maybe(a[3]);
        const double eps = real(a[2]);
        no_tangent("rms_norm", {&x, w, r});
        on_gpu(x);
        if (at::GradMode::is_enabled() && (wants(&x) || wants(w) || wants(r))) {
            const variable_list o = RmsNorm::apply(x, w ? Maybe(*w) : Maybe(), eps, r ? Maybe(*r) : Maybe());
            return r ? tuple(o[0], o[1]) : wrap(o[0]);
        }
        at::AutoDispatchBelowADInplaceOrView below;
        const Normed o = rms_fwd(x, w, eps, r, true, false, -1);
        return r ? tuple(o.y, o.h) : wrap(o.y);
    });
}
// rms_norm_f8(x, weight, eps, residual, format) -> (data, scale, h); h is None without a residual
PyObject *py_rms_norm_f8(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 5, [&] {
        const Normed o = rms_fwd(need(a[0]), maybe(a[1]), real(a[2]), maybe(a[3]), false, false, (int)number(a[4]));
        return tuple(o.q.data, o.q.scale, o.h);
    });
}

// clip(tensors, out or None, p, max_norm or None) -> norm.  max_norm None: the norm alone.
PyObject *py_clip(PyObject *, Args a, Py_ssize_t n)
{
    return guarded(n, 4, [&] {
        if (!PyList_Check(a[0])) fail(PyExc_TypeError, "expected a list of tensors");
        const Py_ssize_t k = PyList_GET_SIZE(a[0]);
        if (k == 0) fail(PyExc_ValueError, "expected at least one tensor");
        const bool clip = a[3] != Py_None, list = clip && PyList_Check(a[1]), flat = clip && !list && a[1] != Py_None;
        if (list && PyList_GET_SIZE(a[1]) != k) fail(PyExc_ValueError, "out must have a tensor for each gradient");
        std::vector<lcf_grad> t((size_t)k);
        const at::Tensor &first = need(PyList_GET_ITEM(a[0], 0));
        const On on(first);
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
                written(o);
            } else if (clip && !flat) {
                written(g);
            }
        }
        if (flat) {
            const at::Tensor &o = take(a[1], "out");
            if (!o.is_contiguous() || o.numel() != total)
                fail(PyExc_ValueError, "out must be a contiguous tensor with as many elements as the gradients have together");
            written(o);
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
                              ws.data_ptr(), (size_t)ws.numel(), on.st));
        else
            check(L.grad_norm(t.data(), (int)k, (int)number(a[2]), (float *)norm.data_ptr(), ws.data_ptr(),
                              (size_t)ws.numel(), on.st));
        return wrap(norm);
    });
}

#define METHOD(name) {#name, (PyCFunction)(void (*)())py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),      METHOD(f8_quant), METHOD(f8_rows),     METHOD(f8_mm), METHOD(f8_product),
                         METHOD(f8_linear), METHOD(rms_norm), METHOD(rms_norm_f8), METHOD(clip),  {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_row_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__row_ops(void) { return PyModule_Create(&module); }
