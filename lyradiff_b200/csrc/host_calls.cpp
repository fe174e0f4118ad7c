// Calls of the FP4, norm and rotary operators over torch tensors: the argument checks, the outputs' allocation and the C-ABI call of one operator in one
// step of host code.  In Python these took 14 to 18 us of a call whose kernel takes 2 to 6 (one token); here 3 to 7, and 11 for a
// norm that writes FP4, its buffers and the product behind it.  The module is bound to the
// functions of the liblyraq.so that the ctypes loader has loaded (bind), so there is one library and one loader.  Functions return what
// lyradiff_b200/ops.py documents; they raise ValueError or TypeError for arguments that do not fit and LyraqError for a status.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <string>
#include <utility>

#include "../../include/lyraq.h"

namespace {

using at::Tensor;

decltype(&lyraq_gated_residual_norm) g_norm        = nullptr;
decltype(&lyraq_rope_axes)           g_rope        = nullptr;
decltype(&lyraq_linear_fp4_forward)  g_linear_fp4  = nullptr;
decltype(&lyraq_gemm_fp4)            g_gemm_fp4    = nullptr;
decltype(&lyraq_quant_fp4)           g_quant_fp4   = nullptr;
decltype(&lyraq_workspace_bytes)     g_workspace   = nullptr;
decltype(&lyraq_fp4_scale_bytes)     g_scale_bytes = nullptr;
PyObject*                            g_error       = nullptr;   // LyraqError(status, where)

// A Python error is set and this is thrown; call() turns it into the function's NULL.
struct Refused {};

[[noreturn]] void refuse(PyObject* type, const char* format, ...)
{
    va_list args;
    va_start(args, format);
    PyErr_FormatV(type, format, args);
    va_end(args);
    throw Refused{};
}

void check_status(int status, const char* where)
{
    if (status != LYRAQ_OK) {
        PyObject* e = PyObject_CallFunction(g_error, "is", status, where);
        if (e != nullptr) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
        throw Refused{};
    }
}

// The tensor behind an argument; null for None.
const Tensor* tensor(PyObject* o, const char* what, int device)
{
    if (o == Py_None) {
        return nullptr;
    }
    if (!THPVariable_Check(o)) {
        refuse(PyExc_TypeError, "%s must be a tensor or None", what);
    }
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != device) {
        refuse(PyExc_ValueError, "%s is on %s, but the current device is cuda:%d", what, t.device().str().c_str(), device);
    }
    return &t;
}

const Tensor& needed(PyObject* o, const char* what, int device)
{
    const Tensor* t = tensor(o, what, device);
    if (t == nullptr) {
        refuse(PyExc_TypeError, "%s must be a tensor", what);
    }
    return *t;
}

void* at_contiguous(const Tensor* t, const char* what)
{
    if (t != nullptr && !t->is_contiguous()) {
        refuse(PyExc_ValueError, "%s must be contiguous", what);
    }
    return t == nullptr ? nullptr : t->data_ptr();
}

int dtype_code(const Tensor& t, const char* what)
{
    switch (t.scalar_type()) {
        case at::kHalf: return LYRAQ_F16;
        case at::kBFloat16: return LYRAQ_BF16;
        case at::kFloat: return LYRAQ_F32;
        default: refuse(PyExc_TypeError, "%s: unsupported dtype %s", what, c10::toString(t.scalar_type()));
    }
}

long as_long(PyObject* o)
{
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        throw Refused{};
    }
    return v;
}

float as_float(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        throw Refused{};
    }
    return (float)v;
}

Tensor empty_like_cuda(at::IntArrayRef sizes, at::ScalarType type, int device)
{
    return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// A result: the argument itself where it was given, else the new tensor.
PyObject* result(PyObject* given, const Tensor& made)
{
    if (given != Py_None) {
        return Py_NewRef(given);
    }
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(Py_None);
}

// A launch may wait for room in the stream, and what holds the stream may be a callback that wants the interpreter.
struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};
template<typename F, typename... A> int run(F* f, A... args)
{
    NoGil free;
    return f(args...);
}

void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// Whether a view may hold one element of memory twice: dimensions by stride, each must step past what lies inside it.
bool overlaps(const Tensor& t)
{
    std::pair<int64_t, int64_t> d[8];
    int                         n = 0;
    for (int64_t i = 0; i < t.dim() && i < 8; ++i) {
        if (t.size(i) > 1) {
            d[n++] = {t.stride(i), t.size(i)};
        }
    }
    std::sort(d, d + n);
    int64_t span = 1;
    for (int i = 0; i < n; ++i) {
        if (d[i].first < span) {
            return true;
        }
        span += d[i].first * (d[i].second - 1);
    }
    return false;
}

// One FP4 matrix: codes uint8 [rows, k / 2], block scales, tensor scale (fp32 [1] or None).  A kernel would read past parts that do not fit.
struct Fp4 {
    uint8_t* codes;
    uint8_t* scales;
    float*   scale;
};
Fp4 fp4_of(PyObject* codes, PyObject* scales, PyObject* scale, int64_t rows, int64_t k, int format, int dev)
{
    const Tensor& c = needed(codes, "FP4 codes", dev);
    const Tensor& s = needed(scales, "FP4 block scales", dev);
    const Tensor* g = tensor(scale, "an FP4 tensor scale", dev);
    if (k % 32 != 0 || c.scalar_type() != at::kByte || c.dim() != 2 || c.size(0) != rows || c.size(1) != k / 2) {
        refuse(PyExc_ValueError, "FP4 codes must be uint8 [%lld, %lld / 2], k a multiple of 32", (long long)rows, (long long)k);
    }
    if (s.scalar_type() != at::kByte || (size_t)s.numel() != g_scale_bytes((size_t)rows, (size_t)k, format)) {
        refuse(PyExc_ValueError, "FP4 block scales do not fit [%lld, %lld]", (long long)rows, (long long)k);
    }
    if (g != nullptr && (g->scalar_type() != at::kFloat || g->numel() != 1)) {
        refuse(PyExc_ValueError, "an FP4 tensor scale is one fp32 number");
    }
    return Fp4{(uint8_t*)at_contiguous(&c, "FP4 codes"), (uint8_t*)at_contiguous(&s, "FP4 block scales"), g == nullptr ? nullptr : (float*)g->data_ptr()};
}

struct Rows {
    void*  p     = nullptr;
    size_t batch = 0, row = 0;
};

// [batch, seq, dim] with contiguous rows; an output's rows must not share memory.
Rows rows_of(const Tensor& t, const char* what, at::IntArrayRef shape, at::ScalarType type, bool output)
{
    if (t.sizes() != shape || t.scalar_type() != type) {
        refuse(PyExc_ValueError, "%s must be [%lld, %lld, %lld] of %s", what, (long long)shape[0], (long long)shape[1], (long long)shape[2], c10::toString(type));
    }
    if (shape[2] > 1 && t.stride(2) != 1) {
        refuse(PyExc_ValueError, "%s: rows must be contiguous", what);
    }
    if (output && !t.is_contiguous() && overlaps(t)) {
        refuse(PyExc_ValueError, "%s has overlapping rows", what);
    }
    return Rows{t.data_ptr(), shape[0] > 1 ? (size_t)t.stride(0) : 0, shape[1] > 1 ? (size_t)t.stride(1) : 0};
}

// (y, x, gate, scale, shift, post_weight, pre_weight, post, pre, residual_scale, eps, x_out, h, qf8, f8_scale, q4 codes, q4 scales,
//  q4 tensor scale, q4 format) -> (x_out, h)
PyObject* gated_residual_norm(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& y   = needed(a[0], "y", dev);
    const Tensor& x   = needed(a[1], "x", dev);
    if (y.dim() != 3) {
        refuse(PyExc_ValueError, "expected [batch, seq, dim]");
    }
    const at::IntArrayRef shape = y.sizes();
    const auto            type  = y.scalar_type();
    lyraq_gated_norm_t    n{};
    n.dtype   = dtype_code(y, "y");
    n.batch   = (size_t)shape[0];
    n.seq_len = (size_t)shape[1];
    n.dim     = (size_t)shape[2];
    n.post    = (int)as_long(a[7]);
    n.pre     = (int)as_long(a[8]);
    n.residual_scale = as_float(a[9]);
    n.eps            = as_float(a[10]);
    const Rows ry = rows_of(y, "y", shape, type, false), rx = rows_of(x, "x", shape, type, false);
    n.y = ry.p; n.y_batch = ry.batch; n.y_row = ry.row;
    n.x = rx.p; n.x_batch = rx.batch; n.x_row = rx.row;
    Tensor        x_new, h_new;
    const Tensor* xo = tensor(a[11], "x_out", dev);
    const Tensor* h  = tensor(a[12], "h", dev);
    const Tensor* q8 = tensor(a[13], "qf8", dev);
    const Tensor* s8 = tensor(a[14], "f8_scale", dev);
    if (q8 != nullptr && (s8 == nullptr || s8->scalar_type() != at::kFloat || s8->numel() != 1 || q8->scalar_type() != at::kByte || q8->numel() != y.numel())) {
        refuse(PyExc_ValueError, "qf8 must be uint8 of y's size, with an fp32 f8_scale");
    }
    auto per_batch = [&](PyObject* o, const char* what, const void*& p, size_t& stride) {
        const Tensor* t = tensor(o, what, dev);
        if (t == nullptr) {
            return;
        }
        const int64_t d = t->dim();
        if (t->scalar_type() != type || d < 1 || d > 2 || t->size(d - 1) != shape[2] || (d == 2 && t->size(0) != shape[0]) ||
            (shape[2] > 1 && t->stride(d - 1) != 1)) {
            refuse(PyExc_ValueError, "%s must be [%lld, %lld] or [%lld] of y's dtype", what, (long long)shape[0], (long long)shape[2], (long long)shape[2]);
        }
        p      = t->data_ptr();
        stride = d == 2 && shape[0] > 1 ? (size_t)t->stride(0) : 0;
    };
    per_batch(a[2], "gate", n.gate, n.gate_batch);
    per_batch(a[3], "scale", n.scale, n.scale_batch);
    per_batch(a[4], "shift", n.shift, n.shift_batch);
    auto weight = [&](PyObject* o, const char* what) -> const void* {
        const Tensor* t = tensor(o, what, dev);
        if (t != nullptr && (t->scalar_type() != type || t->dim() != 1 || t->size(0) != shape[2])) {
            refuse(PyExc_ValueError, "%s must be [%lld] of y's dtype", what, (long long)shape[2]);
        }
        return at_contiguous(t, what);
    };
    n.post_weight = weight(a[5], "post_weight");
    n.pre_weight  = weight(a[6], "pre_weight");
    n.qf8         = (uint8_t*)at_contiguous(q8, "qf8");
    n.f8_scale    = q8 == nullptr ? nullptr : (const float*)s8->data_ptr();
    if (a[15] != Py_None) {
        n.q4_format       = (int)as_long(a[18]);
        const Fp4 q4      = fp4_of(a[15], a[16], a[17], shape[0] * shape[1], shape[2], n.q4_format, dev);
        n.q4              = q4.codes;
        n.q4_scales       = q4.scales;
        n.q4_tensor_scale = q4.scale;
    }
    // rows of a new output are contiguous
    auto output = [&](const Tensor* given, const char* what, Tensor& made, void*& p, size_t& batch, size_t& row) {
        if (given == nullptr) {
            made = empty_like_cuda(shape, type, dev);
        }
        const Rows r = rows_of(given == nullptr ? made : *given, what, shape, type, true);
        p = r.p; batch = r.batch; row = r.row;
    };
    output(xo, "x_out", x_new, n.x_out, n.x_out_batch, n.x_out_row);
    if (h != nullptr || (q8 == nullptr && n.q4 == nullptr)) {
        output(h, "h", h_new, n.h, n.h_batch, n.h_row);
    }
    check_status(run(g_norm, &n, current_stream()), "lyraq_gated_residual_norm");
    return Py_BuildValue("(NN)", result(a[11], x_new), result(a[12], h_new));
}

// (turns, axis, pairs, axes, interleaved, positions, q, k, q_norm, k_norm, eps, q_out, k_out) -> (q_out, k_out)
PyObject* rope_axes(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& q   = needed(a[6], "q", dev);
    if (q.dim() != 4) {
        refuse(PyExc_ValueError, "expected q [batch, seq, heads, head_dim]");
    }
    const int64_t     batch = q.size(0), seq = q.size(1), dim = q.size(3);
    const auto        type = q.scalar_type();
    lyraq_rope_axes_t r{};
    r.dtype       = dtype_code(q, "q");
    r.batch       = (size_t)batch;
    r.seq_len     = (size_t)seq;
    r.head_dim    = (int)std::min<int64_t>(dim, 0x7fffffff);
    r.pairs       = (int)as_long(a[2]);
    const long axes = as_long(a[3]);
    r.interleaved = (int)as_long(a[4]);
    r.eps         = as_float(a[10]);
    const Tensor& turns = needed(a[0], "the plan", dev);
    const Tensor& axis  = needed(a[1], "the plan", dev);
    if (turns.scalar_type() != at::kLong || axis.scalar_type() != at::kByte || turns.numel() != r.pairs || axis.numel() != r.pairs) {
        refuse(PyExc_ValueError, "the plan must be int64 and uint8 of its pairs");
    }
    r.turns = (const uint64_t*)at_contiguous(&turns, "the plan");
    r.axis  = (const unsigned char*)at_contiguous(&axis, "the plan");

    const Tensor& pos = needed(a[5], "positions", dev);
    const int64_t pd  = pos.dim();
    switch (pos.scalar_type()) {
        case at::kInt: r.pos_dtype = LYRAQ_S32; break;
        case at::kLong: r.pos_dtype = LYRAQ_S64; break;
        case at::kFloat: r.pos_dtype = LYRAQ_F32; break;
        default: refuse(PyExc_TypeError, "positions must be int32, int64 or fp32");
    }
    if (pd < 2 || pd > 3 || pos.size(pd - 1) != axes || pos.size(pd - 2) != seq || (pd == 3 && pos.size(0) != batch)) {
        refuse(PyExc_ValueError, "positions must be [%lld, %lld, %ld] or [%lld, %ld]", (long long)batch, (long long)seq, axes, (long long)seq, axes);
    }
    r.positions = pos.data_ptr();
    r.pos_batch = pd == 3 ? (size_t)pos.stride(0) : 0;
    r.pos_token = (size_t)pos.stride(pd - 2);
    r.pos_axis  = (size_t)pos.stride(pd - 1);

    Tensor made[2];
    auto heads = [&](PyObject* in, PyObject* out, PyObject* norm, int i, const void*& p, size_t& pb, size_t& pt, size_t& ph, void*& o, size_t& ob, size_t& ot,
                     size_t& oh, const void*& w, int& count) {
        const char*   name = i == 0 ? "q" : "k";
        const Tensor* t    = tensor(in, name, dev);
        if (t == nullptr) {
            if (out != Py_None || norm != Py_None) {
                refuse(PyExc_ValueError, "an output or a norm of %s without it", name);
            }
            return;
        }
        if (t->dim() != 4 || t->size(0) != batch || t->size(1) != seq || t->size(3) != dim || t->scalar_type() != type) {
            refuse(PyExc_ValueError, "%s must be [%lld, %lld, heads, %lld] of q's dtype", name, (long long)batch, (long long)seq, (long long)dim);
        }
        const Tensor* g = tensor(out, name, dev);
        if (g == nullptr) {
            made[i] = empty_like_cuda(t->sizes(), type, dev);
            g       = &made[i];
        } else if (g->sizes() != t->sizes() || g->scalar_type() != type) {
            refuse(PyExc_ValueError, "the output of %s must have its shape and dtype", name);
        } else if (!g->is_contiguous() && overlaps(*g)) {
            refuse(PyExc_ValueError, "the output of %s has overlapping elements", name);
        }
        if (dim > 1 && (t->stride(3) != 1 || g->stride(3) != 1)) {
            refuse(PyExc_ValueError, "%s: heads must be contiguous", name);
        }
        const Tensor* n = tensor(norm, "a norm's weights", dev);
        if (n != nullptr && (n->scalar_type() != type || n->dim() != 1 || n->size(0) != dim)) {
            refuse(PyExc_ValueError, "the norm weights of %s must be [%lld] of q's dtype", name, (long long)dim);
        }
        auto stride = [](const Tensor& v, int64_t d) { return v.size(d) > 1 ? (size_t)v.stride(d) : 0; };   // of a dimension of one: anything
        p = t->data_ptr(); pb = stride(*t, 0); pt = stride(*t, 1); ph = stride(*t, 2);
        o = g->data_ptr(); ob = stride(*g, 0); ot = stride(*g, 1); oh = stride(*g, 2);
        w     = at_contiguous(n, "a norm's weights");
        count = (int)std::min<int64_t>(t->size(2), 0x7fffffff);
    };
    heads(a[6], a[11], a[8], 0, r.q, r.q_batch, r.q_token, r.q_head, r.q_out, r.q_out_batch, r.q_out_token, r.q_out_head, r.q_norm, r.q_heads);
    heads(a[7], a[12], a[9], 1, r.k, r.k_batch, r.k_token, r.k_head, r.k_out, r.k_out_batch, r.k_out_token, r.k_out_head, r.k_norm, r.k_heads);
    check_status(run(g_rope, &r, current_stream()), "lyraq_rope_axes");
    return Py_BuildValue("(NN)", result(a[11], made[0]), result(a[12], made[1]));
}

void check_epilogue(const Tensor* bias, const Tensor* residual, at::ScalarType type, int64_t m, int64_t n)
{
    if (bias != nullptr && (bias->scalar_type() != type || bias->numel() != n)) {
        refuse(PyExc_ValueError, "bias must be [%lld] of the output's dtype", (long long)n);
    }
    if (residual != nullptr && (residual->scalar_type() != type || residual->dim() < 1 || residual->numel() != m * n || residual->size(residual->dim() - 1) != n)) {
        refuse(PyExc_ValueError, "residual must be [%lld, %lld] of the output's dtype", (long long)m, (long long)n);
    }
}

int as_size(int64_t v, const char* what)
{
    if (v < 0 || v > 0x7fffffff) {
        refuse(PyExc_ValueError, "%s is out of range", what);
    }
    return (int)v;
}

// (x, codes, scales, tensor scale of the weight, n, k, format, input scale, bias, residual, beta, epilogue, out) -> y
PyObject* linear_fp4(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& x   = needed(a[0], "x", dev);
    const int     n = as_size(as_long(a[4]), "n"), k = as_size(as_long(a[5]), "k"), format = (int)as_long(a[6]);
    if (x.dim() < 1 || x.size(x.dim() - 1) != k || k == 0) {
        refuse(PyExc_ValueError, "expected [..., %d]", k);
    }
    const auto type = x.scalar_type();
    const int  m    = as_size(x.numel() / k, "the number of rows");
    const Fp4  w    = fp4_of(a[1], a[2], a[3], n, k, format, dev);
    const Tensor* g = tensor(a[7], "input_scale", dev);
    if (g != nullptr && (g->scalar_type() != at::kFloat || g->numel() != 1)) {
        refuse(PyExc_ValueError, "input_scale is one fp32 number");
    }
    const Tensor* bias     = tensor(a[8], "bias", dev);
    const Tensor* residual = tensor(a[9], "residual", dev);
    check_epilogue(bias, residual, type, m, n);
    // rows that lie one pitch apart stay where they are
    Tensor flat;
    size_t ldx = (size_t)k;
    if (!x.is_contiguous()) {
        flat = x.reshape({m, k});
        ldx  = m > 1 ? (size_t)flat.stride(0) : (size_t)k;
        if ((k > 1 && flat.stride(1) != 1) || (m > 1 && flat.stride(0) < k)) {
            flat = flat.contiguous();
            ldx  = (size_t)k;
        }
    }
    const Tensor* out = tensor(a[12], "out", dev);
    if (out != nullptr && (out->scalar_type() != type || out->dim() < 1 || out->numel() != (int64_t)m * n || out->size(out->dim() - 1) != n)) {
        refuse(PyExc_ValueError, "out must be [..., %d] of x's dtype", n);
    }
    Tensor y;
    if (out == nullptr) {
        c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = n;
        y            = empty_like_cuda(sizes, type, dev);
        out          = &y;
    }
    const size_t need = g_workspace(LYRAQ_OP_LINEAR_FP4, m, n, k);
    const Tensor ws   = empty_like_cuda({(int64_t)need}, at::kByte, dev);
    void* const  yp   = at_contiguous(out, "out");
    const void*  bp   = at_contiguous(bias, "bias");
    const void*  rp   = at_contiguous(residual, "residual");
    check_status(run(g_linear_fp4, yp, (flat.defined() ? flat : x).data_ptr(), dtype_code(x, "x"), ldx, g == nullptr ? nullptr : (const float*)g->data_ptr(),
                     w.codes, w.scales, w.scale, format, bp, rp, as_float(a[10]), (int)as_long(a[11]), m, n, k, ws.data_ptr(), need, current_stream()),
                 "lyraq_linear_fp4_forward");
    return result(a[12], y);
}

// (codes, scales, tensor scale of X, rows, the same of W, k, format, bias, residual, beta, epilogue, Y or the dtype of a new one) -> Y
PyObject* gemm_fp4(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const int     m = as_size(as_long(a[3]), "m"), n = as_size(as_long(a[7]), "n"), k = as_size(as_long(a[8]), "k"), format = (int)as_long(a[9]);
    const Fp4     x = fp4_of(a[0], a[1], a[2], m, k, format, dev), w = fp4_of(a[4], a[5], a[6], n, k, format, dev);
    Tensor        made;
    if (THPDtype_Check(a[14])) {
        const at::ScalarType type = reinterpret_cast<THPDtype*>(a[14])->scalar_type;
        if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) {
            refuse(PyExc_TypeError, "Y: unsupported dtype %s", c10::toString(type));
        }
        made = empty_like_cuda({m, n}, type, dev);
    }
    const Tensor& y = made.defined() ? made : needed(a[14], "Y", dev);
    if (y.dim() != 2 || y.size(0) != m || y.size(1) != n) {
        refuse(PyExc_ValueError, "Y must be [%d, %d]", m, n);
    }
    const Tensor* bias     = tensor(a[10], "bias", dev);
    const Tensor* residual = tensor(a[11], "residual", dev);
    check_epilogue(bias, residual, y.scalar_type(), m, n);
    void* const yp = at_contiguous(&y, "Y");
    const void* bp = at_contiguous(bias, "bias");
    const void* rp = at_contiguous(residual, "residual");
    check_status(run(g_gemm_fp4, x.codes, x.scales, x.scale, w.codes, w.scales, w.scale, format, yp, dtype_code(y, "Y"), bp, rp, as_float(a[12]),
                     (int)as_long(a[13]), m, n, k, current_stream()),
                 "lyraq_gemm_fp4");
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(a[14]);
}

// (rows, k, format, device) -> (codes, scales) of an FP4 matrix
PyObject* fp4_empty(PyObject* const* a)
{
    const int rows = as_size(as_long(a[0]), "rows"), k = as_size(as_long(a[1]), "k"), format = (int)as_long(a[2]), dev = as_size(as_long(a[3]), "the device");
    const Tensor codes  = empty_like_cuda({rows, k / 2}, at::kByte, dev);
    const Tensor scales = empty_like_cuda({(int64_t)g_scale_bytes((size_t)rows, (size_t)k, format)}, at::kByte, dev);
    return Py_BuildValue("(NN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales));
}

// (x, codes, scales, tensor scale, format)
PyObject* quant_fp4(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& x   = needed(a[0], "x", dev);
    if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1))) {
        refuse(PyExc_ValueError, "expected a matrix with contiguous rows that do not overlap");
    }
    const int format = (int)as_long(a[4]);
    const Fp4 q      = fp4_of(a[1], a[2], a[3], x.size(0), x.size(1), format, dev);
    check_status(run(g_quant_fp4, q.codes, q.scales, x.data_ptr(), dtype_code(x, "x"), x.size(0) > 1 ? (size_t)x.stride(0) : (size_t)x.size(1), q.scale,
                     format, (size_t)x.size(0), (size_t)x.size(1), current_stream()),
                 "lyraq_quant_fp4");
    Py_RETURN_NONE;
}

template<PyObject* (*F)(PyObject* const*), Py_ssize_t COUNT> PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != COUNT) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", COUNT, n);
        return nullptr;
    }
    if (g_error == nullptr) {
        PyErr_SetString(PyExc_RuntimeError, "not bound to liblyraq.so");
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ({function name: address}, LyraqError)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    if (n != 2 || !PyDict_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "bind(addresses, error)");
        return nullptr;
    }
    auto take = [&](const char* name, auto& f) {
        PyObject* v = PyDict_GetItemString(args[0], name);
        void*     p = v == nullptr ? nullptr : PyLong_AsVoidPtr(v);
        if (p == nullptr && !PyErr_Occurred()) {
            PyErr_Format(PyExc_ValueError, "no address of %s", name);
        }
        f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
        return p != nullptr;
    };
    if (!take("lyraq_gated_residual_norm", g_norm) || !take("lyraq_rope_axes", g_rope) || !take("lyraq_linear_fp4_forward", g_linear_fp4) ||
        !take("lyraq_gemm_fp4", g_gemm_fp4) || !take("lyraq_quant_fp4", g_quant_fp4) || !take("lyraq_workspace_bytes", g_workspace) ||
        !take("lyraq_fp4_scale_bytes", g_scale_bytes)) {
        return nullptr;
    }
    Py_XSETREF(g_error, Py_NewRef(args[1]));
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {"gated_residual_norm", (PyCFunction)(void (*)())call<gated_residual_norm, 19>, METH_FASTCALL, nullptr},
    {"rope_axes", (PyCFunction)(void (*)())call<rope_axes, 13>, METH_FASTCALL, nullptr},
    {"linear_fp4", (PyCFunction)(void (*)())call<linear_fp4, 13>, METH_FASTCALL, nullptr},
    {"gemm_fp4", (PyCFunction)(void (*)())call<gemm_fp4, 15>, METH_FASTCALL, nullptr},
    {"fp4_empty", (PyCFunction)(void (*)())call<fp4_empty, 4>, METH_FASTCALL, nullptr},
    {"quant_fp4", (PyCFunction)(void (*)())call<quant_fp4, 5>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", "Native calls of lyradiff_b200.ops.", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&g_module); }
