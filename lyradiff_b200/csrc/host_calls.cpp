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
decltype(&lyraq_linear_fp8_block_forward) g_linear_fp8_block = nullptr;
decltype(&lyraq_gemm_fp8_block)      g_gemm_fp8_block  = nullptr;
decltype(&lyraq_quant_fp8_block)     g_quant_fp8_block = nullptr;
decltype(&lyraq_block_means)         g_block_means  = nullptr;
decltype(&lyraq_select_blocks)       g_select       = nullptr;
decltype(&lyraq_select_blocks_workspace) g_select_ws = nullptr;
decltype(&lyraq_sparse_attention)    g_sparse       = nullptr;
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

// The rows [m, k] of a linear's input: rows that lie one pitch apart stay where they are.
const void* flat_rows(const Tensor& x, int m, int k, Tensor& flat, size_t& ldx)
{
    ldx = (size_t)k;
    if (x.is_contiguous()) {
        return x.data_ptr();
    }
    flat = x.reshape({m, k});
    ldx  = m > 1 ? (size_t)flat.stride(0) : (size_t)k;
    if ((k > 1 && flat.stride(1) != 1) || (m > 1 && flat.stride(0) < k)) {
        flat = flat.contiguous();
        ldx  = (size_t)k;
    }
    return flat.data_ptr();
}

// The result of a linear: the argument, or a new tensor.
const Tensor& linear_out(PyObject* o, const Tensor& x, int m, int n, Tensor& made, int dev)
{
    const Tensor* out = tensor(o, "out", dev);
    if (out != nullptr) {
        if (out->scalar_type() != x.scalar_type() || out->dim() < 1 || out->numel() != (int64_t)m * n || out->size(out->dim() - 1) != n) {
            refuse(PyExc_ValueError, "out must be [..., %d] of x's dtype", n);
        }
        return *out;
    }
    c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = n;
    made         = empty_like_cuda(sizes, x.scalar_type(), dev);
    return made;
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
    Tensor        flat, made;
    size_t        ldx;
    const void*   xp  = flat_rows(x, m, k, flat, ldx);
    const Tensor& out = linear_out(a[12], x, m, n, made, dev);
    const size_t need = g_workspace(LYRAQ_OP_LINEAR_FP4, m, n, k);
    const Tensor ws   = empty_like_cuda({(int64_t)need}, at::kByte, dev);
    void* const  yp   = at_contiguous(&out, "out");
    const void*  bp   = at_contiguous(bias, "bias");
    const void*  rp   = at_contiguous(residual, "residual");
    check_status(run(g_linear_fp4, yp, xp, dtype_code(x, "x"), ldx, g == nullptr ? nullptr : (const float*)g->data_ptr(),
                     w.codes, w.scales, w.scale, format, bp, rp, as_float(a[10]), (int)as_long(a[11]), m, n, k, ws.data_ptr(), need, current_stream()),
                 "lyraq_linear_fp4_forward");
    return result(a[12], made);
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

// A weight in FP8 with block scales: codes uint8 [n, k], scales fp32 [ceil(n / 128), ceil(k / 128)].
std::pair<const uint8_t*, const float*> fp8_block_weight(PyObject* codes, PyObject* scales, int n, int k, int dev)
{
    const Tensor& c = needed(codes, "the weight's codes", dev);
    const Tensor& s = needed(scales, "the weight's scales", dev);
    if (c.scalar_type() != at::kByte || c.dim() != 2 || c.size(0) != n || c.size(1) != k) {
        refuse(PyExc_ValueError, "the weight's codes must be uint8 [%d, %d]", n, k);
    }
    if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != ((int64_t)n + 127) / 128 || s.size(1) != ((int64_t)k + 127) / 128) {
        refuse(PyExc_ValueError, "the weight's scales must be fp32, one for each 128 x 128 of [%d, %d]", n, k);
    }
    return {(const uint8_t*)at_contiguous(&c, "the weight's codes"), (const float*)at_contiguous(&s, "the weight's scales")};
}

// Scales of rows in FP8, fp32 [rows, ceil(k / 128)] of any steps; the step of a dimension of one is of no use.
const Tensor& fp8_block_scales(PyObject* o, int64_t rows, int64_t k, int dev, size_t& row_step, size_t& block_step)
{
    const Tensor& s = needed(o, "the scales", dev);
    if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != rows || s.size(1) != (k + 127) / 128) {
        refuse(PyExc_ValueError, "the scales must be fp32, one for each 128 values of a row of [%lld, %lld]", (long long)rows, (long long)k);
    }
    row_step   = s.size(0) > 1 ? (size_t)s.stride(0) : 0;
    block_step = s.size(1) > 1 ? (size_t)s.stride(1) : 0;
    return s;
}

// (x, codes, scales of the weight, n, k, bias, residual, beta, epilogue, out) -> y
PyObject* linear_fp8_block(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& x   = needed(a[0], "x", dev);
    const int     n = as_size(as_long(a[3]), "n"), k = as_size(as_long(a[4]), "k");
    if (x.dim() < 1 || x.size(x.dim() - 1) != k || k == 0) {
        refuse(PyExc_ValueError, "expected [..., %d]", k);
    }
    const int  m = as_size(x.numel() / k, "the number of rows");
    const auto w = fp8_block_weight(a[1], a[2], n, k, dev);
    const Tensor* bias     = tensor(a[5], "bias", dev);
    const Tensor* residual = tensor(a[6], "residual", dev);
    check_epilogue(bias, residual, x.scalar_type(), m, n);
    Tensor        flat, made;
    size_t        ldx;
    const void*   xp   = flat_rows(x, m, k, flat, ldx);
    const Tensor& out  = linear_out(a[9], x, m, n, made, dev);
    const size_t  need = g_workspace(LYRAQ_OP_LINEAR_FP8_BLOCK, m, n, k);
    const Tensor  ws   = empty_like_cuda({(int64_t)need}, at::kByte, dev);
    void* const   yp   = at_contiguous(&out, "out");
    const void*   bp   = at_contiguous(bias, "bias");
    const void*   rp   = at_contiguous(residual, "residual");
    check_status(run(g_linear_fp8_block, yp, xp, dtype_code(x, "x"), ldx, w.first, w.second, bp, rp, as_float(a[7]), (int)as_long(a[8]), m, n, k,
                     ws.data_ptr(), need, current_stream()),
                 "lyraq_linear_fp8_block_forward");
    return result(a[9], made);
}

// (codes, scales of X, the same of W, bias, residual, beta, epilogue, Y or the dtype of a new one) -> Y
PyObject* gemm_fp8_block(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& x   = needed(a[0], "X", dev);
    const Tensor& wc  = needed(a[2], "W", dev);
    if (x.scalar_type() != at::kByte || x.dim() != 2 || wc.dim() != 2 || wc.size(1) != x.size(1)) {
        refuse(PyExc_ValueError, "expected codes X uint8 [m, k] and W uint8 [n, k]");
    }
    const int m = as_size(x.size(0), "m"), n = as_size(wc.size(0), "n"), k = as_size(x.size(1), "k");
    size_t        row_step, block_step;
    const Tensor& xs = fp8_block_scales(a[1], m, k, dev, row_step, block_step);
    const auto    w  = fp8_block_weight(a[2], a[3], n, k, dev);
    Tensor        made;
    if (THPDtype_Check(a[8])) {
        const at::ScalarType type = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
        if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) {
            refuse(PyExc_TypeError, "Y: unsupported dtype %s", c10::toString(type));
        }
        made = empty_like_cuda({m, n}, type, dev);
    }
    const Tensor& y = made.defined() ? made : needed(a[8], "Y", dev);
    if (y.dim() != 2 || y.size(0) != m || y.size(1) != n) {
        refuse(PyExc_ValueError, "Y must be [%d, %d]", m, n);
    }
    const Tensor* bias     = tensor(a[4], "bias", dev);
    const Tensor* residual = tensor(a[5], "residual", dev);
    check_epilogue(bias, residual, y.scalar_type(), m, n);
    const uint8_t* xp = (const uint8_t*)at_contiguous(&x, "X");
    void* const    yp = at_contiguous(&y, "Y");
    const void*    bp = at_contiguous(bias, "bias");
    const void*    rp = at_contiguous(residual, "residual");
    check_status(run(g_gemm_fp8_block, xp, (const float*)xs.data_ptr(), row_step, block_step, w.first, w.second, yp, dtype_code(y, "Y"), bp, rp,
                     as_float(a[6]), (int)as_long(a[7]), m, n, k, current_stream()),
                 "lyraq_gemm_fp8_block");
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(a[8]);
}

// (x, codes, scales)
PyObject* quant_fp8_block(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& x   = needed(a[0], "x", dev);
    if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1))) {
        refuse(PyExc_ValueError, "expected a matrix with contiguous rows that do not overlap");
    }
    const Tensor& q = needed(a[1], "codes", dev);
    if (q.scalar_type() != at::kByte || q.sizes() != x.sizes()) {
        refuse(PyExc_ValueError, "codes must be uint8 of x's shape");
    }
    size_t        row_step, block_step;
    const Tensor& s = fp8_block_scales(a[2], x.size(0), x.size(1), dev, row_step, block_step);
    check_status(run(g_quant_fp8_block, (uint8_t*)at_contiguous(&q, "codes"), (float*)s.data_ptr(), row_step, block_step, x.data_ptr(), dtype_code(x, "x"),
                     x.size(0) > 1 ? (size_t)x.stride(0) : (size_t)x.size(1), (size_t)x.size(0), (size_t)x.size(1), current_stream()),
                 "lyraq_quant_fp8_block");
    Py_RETURN_NONE;
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

// ------------------------------------------------------------------------------- attention over selected key blocks
size_t step_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? (size_t)t.stride(d) : 0; }   // of a dimension of one: anything

// int32 [batch] or None
const int* per_sequence(PyObject* o, const char* what, int64_t batch, int dev)
{
    const Tensor* t = tensor(o, what, dev);
    if (t != nullptr && (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != batch)) {
        refuse(PyExc_ValueError, "%s must be int32 [%lld]", what, (long long)batch);
    }
    return (const int*)at_contiguous(t, what);
}

// q, k, v or out: [batch, tokens, heads, head_dim] with contiguous heads
const Tensor& tokens_of(const Tensor& t, const char* what)
{
    if (t.dim() != 4) {
        refuse(PyExc_ValueError, "%s must be [batch, tokens, heads, head_dim]", what);
    }
    if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16) {
        refuse(PyExc_TypeError, "%s: unsupported dtype %s", what, c10::toString(t.scalar_type()));
    }
    if (t.size(3) > 1 && t.stride(3) != 1) {
        refuse(PyExc_ValueError, "%s: heads must be contiguous", what);
    }
    return t;
}

int as_block(PyObject* o)
{
    const int block = as_size(as_long(o), "the block");
    if (block == 0) {
        refuse(PyExc_ValueError, "a block has one token or more");
    }
    return block;
}

int64_t blocks_of(int64_t n, int block) { return (n + block - 1) / block; }

constexpr int kQueryBlock = 128;

// Means of the blocks of x, into `out` or a new tensor.
Tensor means_of(const Tensor& x, int block, const int* lens, const Tensor* out, int newest, int dev)
{
    const int64_t batch = x.size(0), tokens = x.size(1), heads = x.size(2), dim = x.size(3), blocks = blocks_of(tokens, block);
    Tensor        made;
    if (out == nullptr) {
        made = empty_like_cuda({batch, heads, blocks, dim}, at::kFloat, dev);
    } else {
        if (out->scalar_type() != at::kFloat || out->sizes() != at::IntArrayRef({batch, heads, blocks, dim})) {
            refuse(PyExc_ValueError, "the means must be fp32 [%lld, %lld, %lld, %lld]", (long long)batch, (long long)heads, (long long)blocks, (long long)dim);
        }
        made = *out;
    }
    float* p = (float*)at_contiguous(&made, "the means");
    check_status(run(g_block_means, p, x.data_ptr(), dtype_code(x, "x"), step_of(x, 0), step_of(x, 1), step_of(x, 2), lens, block, newest, (size_t)batch,
                     (size_t)tokens, as_size(heads, "the number of heads"), as_size(dim, "head_dim"), current_stream()),
                 "lyraq_block_means");
    return made;
}

// (x, block, lens, out, newest) -> means
PyObject* block_means(PyObject* const* a)
{
    const int     dev  = c10::cuda::current_device();
    const Tensor& x    = tokens_of(needed(a[0], "x", dev), "x");
    const int*    lens = per_sequence(a[2], "lens", x.size(0), dev);
    const Tensor* out  = tensor(a[3], "out", dev);
    const int     n    = as_size(as_long(a[4]), "newest");
    if (n > 0 && out == nullptr) {
        refuse(PyExc_ValueError, "the newest tokens' blocks are written into means that are there (out)");
    }
    const Tensor means = means_of(x, as_block(a[1]), lens, out, n, dev);
    return result(a[3], means);
}

struct Choice {
    int  block, count, sink, window;
    bool shared, causal;
};
Choice choice_of(PyObject* const* a)     // block, count, sink, window, shared, causal
{
    Choice c{as_block(a[0]), as_size(as_long(a[1]), "count"), as_size(as_long(a[2]), "sink"), as_size(as_long(a[3]), "window"), PyObject_IsTrue(a[4]) == 1,
             PyObject_IsTrue(a[5]) == 1};
    if (c.count == 0) {
        refuse(PyExc_ValueError, "count must be positive");
    }
    return c;
}

// Of each sequence, int32 [batch] or null.
struct Lengths {
    const int *k_lens, *q_lens, *q_start;
};
Lengths lengths_of(PyObject* k_lens, PyObject* q_lens, PyObject* q_start, int64_t batch, int dev)
{
    return {per_sequence(k_lens, "k_lens", batch, dev), per_sequence(q_lens, "q_lens", batch, dev), per_sequence(q_start, "q_start", batch, dev)};
}

std::pair<Tensor, Tensor> select_of(const Tensor& qm, const Tensor& km, const Choice& c, int64_t queries, int64_t keys, const Lengths& n, int dev)
{
    const int64_t batch = qm.size(0), heads = qm.size(1), dim = qm.size(3), k_heads = km.size(1), q_blocks = blocks_of(queries, kQueryBlock);
    if (k_heads == 0 || heads % k_heads != 0) {
        refuse(PyExc_ValueError, "the query heads must be a multiple of the key heads");
    }
    const int64_t lists  = c.shared ? k_heads : heads;
    const Tensor  index  = empty_like_cuda({batch, lists, q_blocks, c.count}, at::kInt, dev);
    const Tensor  counts = empty_like_cuda({batch, lists, q_blocks}, at::kInt, dev);
    const size_t  need   = g_select_ws((size_t)batch, (int)lists, (size_t)queries, (size_t)keys, c.block);
    const Tensor  ws     = empty_like_cuda({(int64_t)need}, at::kByte, dev);
    lyraq_select_blocks_t s{};
    s.q_means  = (const float*)at_contiguous(&qm, "q_means");
    s.k_means  = (const float*)at_contiguous(&km, "k_means");
    s.index    = (int*)index.data_ptr();
    s.counts   = (int*)counts.data_ptr();
    s.k_lens   = n.k_lens;
    s.q_lens   = n.q_lens;
    s.q_start  = n.q_start;
    s.batch    = (size_t)batch;
    s.queries  = (size_t)queries;
    s.keys     = (size_t)keys;
    s.q_heads  = as_size(heads, "the number of heads");
    s.k_heads  = as_size(k_heads, "the number of heads");
    s.lists    = (int)lists;
    s.head_dim = as_size(dim, "head_dim");
    s.block    = c.block;
    s.count    = c.count;
    s.sink     = c.sink;
    s.window   = c.window;
    s.causal   = c.causal;
    check_status(run(g_select, &s, ws.data_ptr(), need, current_stream()), "lyraq_select_blocks");
    return {index, counts};
}

// (q_means, k_means, block, count, sink, window, shared, causal, queries, keys, k_lens, q_start, q_lens) -> (index, counts)
PyObject* select_blocks(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& qm  = needed(a[0], "q_means", dev);
    const Tensor& km  = needed(a[1], "k_means", dev);
    const Choice  c   = choice_of(a + 2);
    const int64_t queries = as_size(as_long(a[8]), "queries"), keys = as_size(as_long(a[9]), "keys");
    if (qm.dim() != 4 || km.dim() != 4 || qm.scalar_type() != at::kFloat || km.scalar_type() != at::kFloat || qm.size(2) != blocks_of(queries, kQueryBlock) ||
        km.size(2) != blocks_of(keys, c.block) || km.size(0) != qm.size(0) || km.size(3) != qm.size(3)) {
        refuse(PyExc_ValueError, "expected q_means fp32 [batch, heads, %lld, head_dim] and k_means [batch, key heads, %lld, head_dim]",
               (long long)blocks_of(queries, kQueryBlock), (long long)blocks_of(keys, c.block));
    }
    const auto s = select_of(qm, km, c, queries, keys, lengths_of(a[10], a[12], a[11], qm.size(0), dev), dev);
    return Py_BuildValue("(NN)", THPVariable_Wrap(s.first), THPVariable_Wrap(s.second));
}

void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v)
{
    if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) {
        refuse(PyExc_ValueError, "k and v must be [%lld, keys, heads, %lld] of q's dtype", (long long)q.size(0), (long long)q.size(3));
    }
    if (k.size(2) == 0 || q.size(2) % k.size(2) != 0) {
        refuse(PyExc_ValueError, "the query heads must be a multiple of the key heads");
    }
}

Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& index, const Tensor& counts, int block, const Lengths& n, bool causal, float scale,
              const Tensor* out, int dev)
{
    const int64_t batch = q.size(0), queries = q.size(1), heads = q.size(2), dim = q.size(3), k_heads = k.size(2), q_blocks = blocks_of(queries, kQueryBlock);
    if (index.scalar_type() != at::kInt || index.dim() != 4 || index.size(0) != batch || (index.size(1) != heads && index.size(1) != k_heads) ||
        index.size(2) != q_blocks) {
        refuse(PyExc_ValueError, "index must be int32 [%lld, %lld or %lld, %lld, count]", (long long)batch, (long long)heads, (long long)k_heads, (long long)q_blocks);
    }
    if (counts.scalar_type() != at::kInt || counts.sizes() != index.sizes().slice(0, 3)) {
        refuse(PyExc_ValueError, "counts must be int32 of index's first three dimensions");
    }
    Tensor made;
    if (out == nullptr) {
        made = empty_like_cuda(q.sizes(), q.scalar_type(), dev);
    } else {
        if (tokens_of(*out, "out").sizes() != q.sizes() || out->scalar_type() != q.scalar_type()) {
            refuse(PyExc_ValueError, "out must have q's shape and dtype");
        }
        if (!out->is_contiguous() && overlaps(*out)) {
            refuse(PyExc_ValueError, "out has overlapping elements");
        }
        made = *out;
    }
    lyraq_sparse_attention_t s{};
    s.q = q.data_ptr(); s.k = k.data_ptr(); s.v = v.data_ptr(); s.out = made.data_ptr();
    s.q_batch = step_of(q, 0); s.q_token = step_of(q, 1); s.q_head = step_of(q, 2);
    s.k_batch = step_of(k, 0); s.k_token = step_of(k, 1); s.k_head = step_of(k, 2);
    s.v_batch = step_of(v, 0); s.v_token = step_of(v, 1); s.v_head = step_of(v, 2);
    s.o_batch = step_of(made, 0); s.o_token = step_of(made, 1); s.o_head = step_of(made, 2);
    s.index    = (const int*)at_contiguous(&index, "index");
    s.counts   = (const int*)at_contiguous(&counts, "counts");
    s.k_lens   = n.k_lens;
    s.q_lens   = n.q_lens;
    s.q_start  = n.q_start;
    s.batch    = (size_t)batch;
    s.queries  = (size_t)queries;
    s.keys     = (size_t)k.size(1);
    s.q_heads  = as_size(heads, "the number of heads");
    s.k_heads  = as_size(k_heads, "the number of heads");
    s.lists    = as_size(index.size(1), "the number of lists");
    s.head_dim = as_size(dim, "head_dim");
    s.block    = block;
    s.count    = as_size(index.size(3), "count");
    s.causal   = causal;
    s.softmax_scale = scale;
    s.dtype    = dtype_code(q, "q");
    check_status(run(g_sparse, &s, current_stream()), "lyraq_sparse_attention");
    return made;
}

// (q, k, v, index, counts, block, k_lens, q_start, causal, softmax scale, out, q_lens) -> out
PyObject* sparse_attention(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& q = tokens_of(needed(a[0], "q", dev), "q");
    const Tensor& k = tokens_of(needed(a[1], "k", dev), "k");
    const Tensor& v = tokens_of(needed(a[2], "v", dev), "v");
    check_qkv(q, k, v);
    const Tensor out = attend(q, k, v, needed(a[3], "index", dev), needed(a[4], "counts", dev), as_block(a[5]), lengths_of(a[6], a[11], a[7], q.size(0), dev),
                              PyObject_IsTrue(a[8]) == 1, as_float(a[9]), tensor(a[10], "out", dev), dev);
    return result(a[10], out);
}

// (q, k, v, block, count, sink, window, shared, causal, softmax scale, k_lens, q_start, k_means, out, q_lens) -> (out, index, counts): means, selection and attention
PyObject* select_and_attend(PyObject* const* a)
{
    const int     dev = c10::cuda::current_device();
    const Tensor& q = tokens_of(needed(a[0], "q", dev), "q");
    const Tensor& k = tokens_of(needed(a[1], "k", dev), "k");
    const Tensor& v = tokens_of(needed(a[2], "v", dev), "v");
    check_qkv(q, k, v);
    const Choice  c     = choice_of(a + 3);
    const Lengths n     = lengths_of(a[10], a[14], a[11], q.size(0), dev);
    const Tensor* given = tensor(a[12], "k_means", dev);
    if (given != nullptr && (given->scalar_type() != at::kFloat || given->sizes() != at::IntArrayRef({k.size(0), k.size(2), blocks_of(k.size(1), c.block), k.size(3)}))) {
        refuse(PyExc_ValueError, "k_means must be fp32 [batch, key heads, %lld, head_dim]", (long long)blocks_of(k.size(1), c.block));
    }
    const Tensor qm = means_of(q, kQueryBlock, n.q_lens, nullptr, 0, dev);
    const Tensor km = given != nullptr ? *given : means_of(k, c.block, n.k_lens, nullptr, 0, dev);
    const auto   s  = select_of(qm, km, c, q.size(1), k.size(1), n, dev);
    const Tensor out = attend(q, k, v, s.first, s.second, c.block, n, c.causal, as_float(a[9]), tensor(a[13], "out", dev), dev);
    return Py_BuildValue("(NNN)", result(a[13], out), THPVariable_Wrap(s.first), THPVariable_Wrap(s.second));
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
        !take("lyraq_linear_fp8_block_forward", g_linear_fp8_block) || !take("lyraq_gemm_fp8_block", g_gemm_fp8_block) ||
        !take("lyraq_quant_fp8_block", g_quant_fp8_block) || !take("lyraq_block_means", g_block_means) || !take("lyraq_select_blocks", g_select) ||
        !take("lyraq_select_blocks_workspace", g_select_ws) || !take("lyraq_sparse_attention", g_sparse) || !take("lyraq_fp4_scale_bytes", g_scale_bytes)) {
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
    {"linear_fp8_block", (PyCFunction)(void (*)())call<linear_fp8_block, 10>, METH_FASTCALL, nullptr},
    {"gemm_fp8_block", (PyCFunction)(void (*)())call<gemm_fp8_block, 9>, METH_FASTCALL, nullptr},
    {"quant_fp8_block", (PyCFunction)(void (*)())call<quant_fp8_block, 3>, METH_FASTCALL, nullptr},
    {"block_means", (PyCFunction)(void (*)())call<block_means, 5>, METH_FASTCALL, nullptr},
    {"select_blocks", (PyCFunction)(void (*)())call<select_blocks, 13>, METH_FASTCALL, nullptr},
    {"sparse_attention", (PyCFunction)(void (*)())call<sparse_attention, 12>, METH_FASTCALL, nullptr},
    {"select_and_attend", (PyCFunction)(void (*)())call<select_and_attend, 15>, METH_FASTCALL, nullptr},
    {"fp4_empty", (PyCFunction)(void (*)())call<fp4_empty, 4>, METH_FASTCALL, nullptr},
    {"quant_fp4", (PyCFunction)(void (*)())call<quant_fp4, 5>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", "Native calls of lyradiff_b200.ops.", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&g_module); }
