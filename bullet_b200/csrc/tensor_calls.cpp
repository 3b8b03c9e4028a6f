// The dense trunk's operators on torch tensors, as a Python module: arguments checked, outputs allocated, the C ABI called on torch's
// current stream.
//
// bullet_b200/ops.py is its public face and documents the calls.  They are here and not there because a call for one position takes the
// GPU 2 to 4 us and a launch the host 3.2: with the checks, allocations and ctypes structures in Python a call took 11 to 21 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/bullet_b200.h"

namespace {

PyObject *library_error = nullptr, *memory_error = nullptr;  // bullet_b200._lib.B200Error, torch.OutOfMemoryError

// What ends a call with a Python exception, which is set already.
struct Raised {};

[[noreturn]] void refuse(const std::string& why) {
    PyErr_SetString(PyExc_ValueError, why.c_str());
    throw Raised{};
}
void check(int rc) {
    if (rc >= 0) return;
    PyObject* e = PyObject_CallFunction(library_error, "is", rc, b200_last_error());
    if (e) {
        PyErr_SetObject(library_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return B200_TYPE_F32;
        case at::kBFloat16: return B200_TYPE_BF16;
        case at::kHalf: return B200_TYPE_F16;
        case at::kFloat8_e4m3fn: return B200_TYPE_E4M3;
        default: return -1;
    }
}
enum Types { kFloats, k16Bits, kCodes };
bool among(at::ScalarType t, Types types) {
    const int k = type_of(t);
    return types == kCodes ? k == B200_TYPE_E4M3 : k == B200_TYPE_BF16 || k == B200_TYPE_F16 || (types == kFloats && k == B200_TYPE_F32);
}

using Tensor = const at::Tensor&;
at::Tensor tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + ": a tensor is wanted");
    Tensor t = THPVariable_Unpack(o);
    // (the outputs have no history: a weight would stay where it is without a word)
    if (t.requires_grad() && at::GradMode::is_enabled())
        refuse(std::string(what) + ": requires a gradient, which these calls do not record: take the *_backward calls, under torch.no_grad() or in an autograd.Function");
    return t;
}
std::optional<at::Tensor> maybe_tensor(PyObject* o, const char* what) {
    if (o == Py_None) return std::nullopt;
    return tensor(o, what);
}
at::ScalarType dtype(PyObject* o, const char* what) {
    if (!THPDtype_Check(o)) refuse(std::string(what) + ": a torch type is wanted");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// The distance of a matrix's rows.
int64_t rows_apart(Tensor t, const char* what) {
    if (t.dim() != 2 || !t.is_cuda()) refuse(std::string(what) + ": a matrix on a CUDA device is wanted");
    const int64_t rows = t.size(0), cols = t.size(1), ld = t.stride(0);
    if (rows > INT32_MAX || cols > INT32_MAX) refuse(std::string(what) + ": too many rows or columns");
    if ((t.stride(1) != 1 && cols > 1) || (ld < cols && rows > 1)) refuse(std::string(what) + ": the elements of a row must be consecutive and rows must not overlap");
    return rows > 1 ? ld : std::max(ld, cols);
}
int64_t matrix(Tensor t, const char* what, Types types) {
    if (!among(t.scalar_type(), types)) refuse(std::string(what) + ": this type is not taken here");
    return rows_apart(t, what);
}
// Of one type and shape, where another matrix is.
int64_t matrix(Tensor t, const char* what, at::ScalarType type, int64_t rows, int64_t cols, Tensor beside) {
    const int64_t ld = rows_apart(t, what);
    if (t.scalar_type() != type) refuse(std::string(what) + ": this type is not taken here");
    if (t.size(0) != rows || t.size(1) != cols)
        refuse(std::string(what) + ": shape (" + std::to_string(t.size(0)) + ", " + std::to_string(t.size(1)) + ") where (" + std::to_string(rows) + ", " + std::to_string(cols) + ") is wanted");
    if (t.device() != beside.device()) refuse(std::string(what) + ": on another device");
    return ld;
}
float* vector(const std::optional<at::Tensor>& t, const char* what, int64_t n, Tensor beside) {
    if (!t) return nullptr;
    if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != n || t->device() != beside.device() || !t->is_contiguous())
        refuse(std::string(what) + ": " + std::to_string(n) + " consecutive fp32 values on the same device are wanted");
    return static_cast<float*>(t->data_ptr());
}
int act_of(PyObject* o) {
    const long act = PyLong_AsLong(o);
    if (act == -1 && PyErr_Occurred()) throw Raised{};
    if (act < B200_ACT_NONE || act > B200_ACT_RELU) refuse("act: " + std::to_string(act) + " names no activation");
    return (int)act;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v != 0;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, Tensor beside) { return at::detail::empty_cuda(shape, type, beside.device(), std::nullopt); }
void* stream_of(Tensor t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int device_of(Tensor t) { return t.device().index(); }
void* at_of(const std::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// A call's workspace; torch's allocator hands it on in the stream's order.
template <class Op>
at::Tensor space(int (*query)(const Op*, int64_t*), Op& op, Tensor beside) {
    int64_t bytes = 0;
    check(query(&op, &bytes));
    if (!bytes) return {};
    at::Tensor s = empty({bytes}, at::kByte, beside);
    op.workspace = s.data_ptr();
    op.workspace_bytes = bytes;
    return s;
}

PyObject* wrapped(const std::optional<at::Tensor>& t) {
    if (t) return THPVariable_Wrap(*t);
    Py_RETURN_NONE;
}
template <size_t N>
PyObject* tuple(const std::optional<at::Tensor> (&t)[N]) {
    PyObject* out = PyTuple_New(N);
    if (!out) throw Raised{};
    for (size_t k = 0; k < N; k++) {
        PyObject* o = wrapped(t[k]);
        if (!o) {
            Py_DECREF(out);
            throw Raised{};
        }
        PyTuple_SET_ITEM(out, k, o);
    }
    return out;
}

// (x, weight, residual, eps, out_dtype) -> (y, scale, total or None, rstd)
PyObject* rms_norm(PyObject* const* a) {
    const at::Tensor x = tensor(a[0], "x");
    const auto weight = maybe_tensor(a[1], "weight"), residual = maybe_tensor(a[2], "residual");
    b200_rms_norm_op op{};
    op.ldx = matrix(x, "x", kFloats);
    const int64_t rows = x.size(0), cols = x.size(1);
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
    const at::ScalarType out = a[4] == Py_None ? x.scalar_type() : dtype(a[4], "out_dtype");
    if (type_of(out) < 0) refuse("out_dtype: this type is not taken here");
    op.weight = vector(weight, "weight", cols, x);
    std::optional<at::Tensor> total, scale;
    if (residual) {
        op.ldr = matrix(*residual, "residual", x.scalar_type(), rows, cols, x);
        op.residual = residual->data_ptr();
        total = empty({rows, cols}, x.scalar_type(), x);
    }
    const at::Tensor y = empty({rows, cols}, out, x), rstd = empty({rows}, at::kFloat, x);
    if (out == at::kFloat8_e4m3fn) scale = empty({rows}, at::kFloat, x);
    op.rows = (int)rows, op.cols = (int)cols, op.x_type = type_of(x.scalar_type()), op.y_type = type_of(out);
    op.lds = op.ldy = cols;
    op.x = x.data_ptr(), op.sum = at_of(total), op.y = y.data_ptr(), op.scale = static_cast<float*>(at_of(scale)), op.rstd = static_cast<float*>(rstd.data_ptr());
    op.eps = (float)eps;
    check(b200_op_rms_norm(device_of(x), stream_of(x), &op));
    return tuple<4>({y, scale, total, rstd});
}

// (dy, total, rstd, weight, dtotal) -> (dx, dweight or None)
PyObject* rms_norm_backward(PyObject* const* a) {
    const at::Tensor dy = tensor(a[0], "dy"), total = tensor(a[1], "total"), rstd = tensor(a[2], "rstd");
    const auto weight = maybe_tensor(a[3], "weight"), dtotal = maybe_tensor(a[4], "dtotal");
    b200_rms_norm_grad_op op{};
    op.lds = matrix(total, "total", kFloats);
    const int64_t rows = total.size(0), cols = total.size(1);
    if (!among(dy.scalar_type(), kFloats)) refuse("dy: this type is not taken here");
    op.lddy = matrix(dy, "dy", dy.scalar_type(), rows, cols, total);
    if (dtotal) op.ldds = matrix(*dtotal, "dtotal", total.scalar_type(), rows, cols, total), op.dsum = dtotal->data_ptr();
    op.rstd = vector(rstd, "rstd", rows, total);
    op.weight = vector(weight, "weight", cols, total);
    const at::Tensor dx = empty({rows, cols}, total.scalar_type(), total);
    std::optional<at::Tensor> dweight;
    if (weight) dweight = empty({cols}, at::kFloat, total);
    op.rows = (int)rows, op.cols = (int)cols, op.x_type = type_of(total.scalar_type()), op.dy_type = type_of(dy.scalar_type());
    op.lddx = cols;
    op.dy = dy.data_ptr(), op.sum = total.data_ptr(), op.dx = dx.data_ptr(), op.dweight = static_cast<float*>(at_of(dweight));
    const at::Tensor held = space(b200_op_rms_norm_backward_workspace, op, total);
    check(b200_op_rms_norm_backward(device_of(total), stream_of(total), &op));
    return tuple<2>({dx, dweight});
}

// (x, act, by_column) -> (codes, scale)
PyObject* pack8(PyObject* const* a) {
    const at::Tensor x = tensor(a[0], "x");
    b200_pack8_op op{};
    op.act = act_of(a[1]);
    op.by_column = truth(a[2]);
    op.ldx = matrix(x, "x", kFloats);
    const int64_t rows = x.size(0), cols = x.size(1);
    const at::Tensor codes = empty({rows, cols}, at::kFloat8_e4m3fn, x), scale = empty({op.by_column ? cols : rows}, at::kFloat, x);
    op.rows = (int)rows, op.cols = (int)cols, op.x_type = type_of(x.scalar_type());
    op.ldq = cols;
    op.x = x.data_ptr(), op.q = codes.data_ptr(), op.scale = static_cast<float*>(scale.data_ptr());
    check(b200_op_pack8(device_of(x), stream_of(x), &op));
    return tuple<2>({codes, scale});
}

// (codes, scale, by_column, dtype) -> values
PyObject* unpack8(PyObject* const* a) {
    const at::Tensor q = tensor(a[0], "packed"), scale = tensor(a[1], "packed's scales");
    b200_unpack8_op op{};
    op.by_column = truth(a[2]);
    op.ldq = matrix(q, "packed", kCodes);
    const int64_t rows = q.size(0), cols = q.size(1);
    op.scale = vector(scale, "packed's scales", op.by_column ? cols : rows, q);
    const at::ScalarType out = dtype(a[3], "dtype");
    if (!among(out, kFloats)) refuse("dtype: this type is not taken here");
    const at::Tensor y = empty({rows, cols}, out, q);
    op.rows = (int)rows, op.cols = (int)cols, op.y_type = type_of(out);
    op.ldy = cols;
    op.q = q.data_ptr(), op.y = y.data_ptr();
    check(b200_op_unpack8(device_of(q), stream_of(q), &op));
    return THPVariable_Wrap(y);
}

// (x, x_scale, w, w_scale, bias, act, residual, out_dtype) -> y; scales: of codes, else None
PyObject* dense(PyObject* const* a) {
    const at::Tensor x = tensor(a[0], "x"), w = tensor(a[2], "w");
    const auto x_scale = maybe_tensor(a[1], "x's scales"), w_scale = maybe_tensor(a[3], "w's scales"), bias = maybe_tensor(a[4], "bias"), residual = maybe_tensor(a[6], "residual");
    if ((bool)x_scale != (bool)w_scale) refuse("x and w: both in 8 bits or neither");
    b200_dense_op op{};
    op.act = act_of(a[5]);
    op.ldx = matrix(x, "x", x_scale ? kCodes : k16Bits);
    const int64_t rows = x.size(0), n_in = x.size(1);
    if (w.dim() != 2) refuse("w: a matrix on a CUDA device is wanted");
    const int64_t n_out = w.size(1);
    op.ldw = matrix(w, "w", x.scalar_type(), n_in, n_out, x);
    op.x_scale = vector(x_scale, "x's scales", rows, x);
    op.w_scale = vector(w_scale, "w's scales", n_out, x);
    const at::ScalarType out = a[7] != Py_None ? dtype(a[7], "out_dtype") : x_scale ? at::kBFloat16 : x.scalar_type();
    if (!among(out, kFloats)) refuse("out_dtype: this type is not taken here");
    op.bias = vector(bias, "bias", n_out, x);
    if (residual) op.ldr = matrix(*residual, "residual", out, rows, n_out, x), op.residual = residual->data_ptr();
    const at::Tensor y = empty({rows, n_out}, out, x);
    op.rows = (int)rows, op.in = (int)n_in, op.out = (int)n_out, op.x_type = type_of(x.scalar_type()), op.y_type = type_of(out);
    op.ldy = n_out;
    op.x = x.data_ptr(), op.w = w.data_ptr(), op.y = y.data_ptr();
    const at::Tensor held = space(b200_op_dense_workspace, op, x);
    check(b200_op_dense(device_of(x), stream_of(x), &op));
    return THPVariable_Wrap(y);
}

// ---- 4 bits

// Rows of codes along `length`, and their scales.
struct Codes4 {
    at::Tensor codes, scale;
    int64_t rows, length, ld;
    const uint8_t* scale_at() const { return static_cast<const uint8_t*>(scale.data_ptr()); }
};
int64_t length_of(PyObject* o, const char* what) {
    const long long n = PyLong_AsLongLong(o);
    if (n == -1 && PyErr_Occurred()) throw Raised{};
    if (n < 0 || n > INT32_MAX) refuse(std::string(what) + ": a length of " + std::to_string(n));
    return n;
}
Codes4 codes4(PyObject* codes, PyObject* scale, PyObject* length, const char* what) {
    Codes4 c{tensor(codes, what), tensor(scale, what), 0, length_of(length, what), 0};
    if (c.codes.scalar_type() != at::kByte) refuse(std::string(what) + ": codes are torch.uint8");
    c.ld = rows_apart(c.codes, what);
    c.rows = c.codes.size(0);
    const int64_t groups = (c.length + 31) / 32;
    if (c.codes.size(1) != groups * 16) refuse(std::string(what) + ": " + std::to_string(groups * 16) + " bytes a row are wanted for a length of " + std::to_string(c.length));
    if (c.rows <= 1 || groups == 0) c.ld = groups * 16;  // (there is no second row)
    if (c.ld % 16 || reinterpret_cast<uintptr_t>(c.codes.data_ptr()) % 16) refuse(std::string(what) + ": rows of codes must start on 16 bytes");
    if (c.scale.scalar_type() != at::kByte || c.scale.dim() != 1 || c.scale.size(0) != B200_FOUR_SCALES(c.rows, c.length) || !c.scale.is_contiguous() ||
        c.scale.device() != c.codes.device() || reinterpret_cast<uintptr_t>(c.scale.data_ptr()) % 16)
        refuse(std::string(what) + ": scales are " + std::to_string(B200_FOUR_SCALES(c.rows, c.length)) + " consecutive torch.uint8 on 16 bytes on the same device");
    return c;
}

// (x, by_column) -> (codes, scale)
PyObject* pack4(PyObject* const* a) {
    const at::Tensor x = tensor(a[0], "x");
    b200_pack4_op op{};
    op.by_column = truth(a[1]);
    op.ldx = matrix(x, "x", kFloats);
    const int64_t rows = op.by_column ? x.size(1) : x.size(0), length = op.by_column ? x.size(0) : x.size(1);
    const at::Tensor codes = empty({rows, (length + 31) / 32 * 16}, at::kByte, x), scale = empty({B200_FOUR_SCALES(rows, length)}, at::kByte, x);
    op.rows = (int)x.size(0), op.cols = (int)x.size(1), op.x_type = type_of(x.scalar_type());
    op.ldq = codes.size(1);
    op.x = x.data_ptr(), op.q = codes.data_ptr(), op.scale = static_cast<uint8_t*>(scale.data_ptr());
    check(b200_op_pack4(device_of(x), stream_of(x), &op));
    return tuple<2>({codes, scale});
}

// (codes, scale, length, by_column, dtype) -> values
PyObject* unpack4(PyObject* const* a) {
    const Codes4 q = codes4(a[0], a[1], a[2], "packed");
    b200_unpack4_op op{};
    op.by_column = truth(a[3]);
    const at::ScalarType out = dtype(a[4], "dtype");
    if (!among(out, kFloats)) refuse("dtype: this type is not taken here");
    const int64_t rows = op.by_column ? q.length : q.rows, cols = op.by_column ? q.rows : q.length;
    const at::Tensor y = empty({rows, cols}, out, q.codes);
    op.rows = (int)rows, op.cols = (int)cols, op.y_type = type_of(out);
    op.ldq = q.ld, op.ldy = cols;
    op.q = q.codes.data_ptr(), op.scale = q.scale_at(), op.y = y.data_ptr();
    check(b200_op_unpack4(device_of(y), stream_of(y), &op));
    return THPVariable_Wrap(y);
}

// (x codes, x scale, x length, w codes, w scale, w length, bias, act, residual, out_dtype) -> y
PyObject* dense4(PyObject* const* a) {
    const auto bias = maybe_tensor(a[6], "bias"), residual = maybe_tensor(a[8], "residual");
    const Codes4 x = codes4(a[0], a[1], a[2], "x"), w = codes4(a[3], a[4], a[5], "w");
    b200_dense4_op op{};
    op.act = act_of(a[7]);
    if (x.length != w.length) refuse("x and w: lengths of " + std::to_string(x.length) + " and " + std::to_string(w.length));
    if (w.codes.device() != x.codes.device()) refuse("w: on another device");
    const at::ScalarType out = a[9] != Py_None ? dtype(a[9], "out_dtype") : at::kBFloat16;
    if (!among(out, kFloats)) refuse("out_dtype: this type is not taken here");
    op.bias = vector(bias, "bias", w.rows, x.codes);
    if (residual) op.ldr = matrix(*residual, "residual", out, x.rows, w.rows, x.codes), op.residual = residual->data_ptr();
    const at::Tensor y = empty({x.rows, w.rows}, out, x.codes);
    op.rows = (int)x.rows, op.in = (int)x.length, op.out = (int)w.rows, op.y_type = type_of(out);
    op.ldx = x.ld, op.ldw = w.ld, op.ldy = w.rows;
    op.x = x.codes.data_ptr(), op.x_scale = x.scale_at(), op.w = w.codes.data_ptr(), op.w_scale = w.scale_at(), op.y = y.data_ptr();
    check(b200_op_dense4(device_of(y), stream_of(y), &op));
    return THPVariable_Wrap(y);
}

// ---- rows named by ids

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}
// Lists of ids, [rows] or [rows][slots].
template <class Op>
at::Tensor lists(PyObject* o, Op& op, Tensor beside) {
    const at::Tensor ids = tensor(o, "ids");
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) refuse("ids: torch.int32 or torch.int64 are wanted");
    if (ids.dim() < 1 || ids.dim() > 2 || ids.device() != beside.device()) refuse("ids: a vector, or a matrix of lists, on the same device is wanted");
    const int64_t rows = ids.size(0), slots = ids.dim() == 2 ? ids.size(1) : 1;
    if (rows > INT32_MAX || slots > INT32_MAX) refuse("ids: too many");
    if (ids.dim() == 2 && slots > 1 && ids.stride(1) != 1) refuse("ids: a list's must be consecutive");
    if (rows > 1 && ids.stride(0) < slots) refuse("ids: lists must not overlap");
    op.rows = (int)rows, op.slots = (int)slots, op.wide_ids = ids.scalar_type() == at::kLong;
    op.ldids = rows > 1 ? ids.stride(0) : slots;
    op.ids = ids.data_ptr();
    return ids;
}

// (table, ids, scale, out_dtype) -> y
PyObject* embed(PyObject* const* a) {
    const at::Tensor table = tensor(a[0], "table");
    b200_embed_op op{};
    op.ldt = matrix(table, "table", kFloats);
    const at::Tensor ids = lists(a[1], op, table);
    op.scale = (float)number(a[2]);
    const at::ScalarType out = a[3] == Py_None ? table.scalar_type() : dtype(a[3], "out_dtype");
    if (!among(out, kFloats)) refuse("out_dtype: this type is not taken here");
    const at::Tensor y = empty({op.rows, table.size(1)}, out, table);
    op.n = (int)table.size(0), op.cols = (int)table.size(1), op.table_type = type_of(table.scalar_type()), op.y_type = type_of(out);
    op.ldy = op.cols;
    op.table = table.data_ptr(), op.y = y.data_ptr();
    check(b200_op_embed(device_of(table), stream_of(table), &op));
    return THPVariable_Wrap(y);
}

// (dy, ids, n, scale, dtype) -> dtable
PyObject* embed_backward(PyObject* const* a) {
    const at::Tensor dy = tensor(a[0], "dy");
    b200_embed_grad_op op{};
    op.lddy = matrix(dy, "dy", kFloats);
    const at::Tensor ids = lists(a[1], op, dy);
    if (ids.size(0) != dy.size(0)) refuse("ids: " + std::to_string(ids.size(0)) + " lists where " + std::to_string(dy.size(0)) + " are wanted");
    const int64_t n = length_of(a[2], "n");
    op.scale = (float)number(a[3]);
    const at::ScalarType out = dtype(a[4], "dtype");
    if (!among(out, kFloats)) refuse("dtype: this type is not taken here");
    const at::Tensor dtable = empty({n, dy.size(1)}, out, dy);
    op.n = (int)n, op.cols = (int)dy.size(1), op.dy_type = type_of(dy.scalar_type()), op.dtable_type = type_of(out);
    op.lddt = op.cols;
    op.dy = dy.data_ptr(), op.dtable = dtable.data_ptr();
    const at::Tensor held = space(b200_op_embed_backward_workspace, op, dy);
    check(b200_op_embed_backward(device_of(dy), stream_of(dy), &op));
    return THPVariable_Wrap(dtable);
}

// ---- the norm of gradients

struct Reference {
    PyObject* o;
    ~Reference() { Py_XDECREF(o); }
};
// Whether the elements of two tensors of one shape lie alike (a dimension of one element lies anyhow, and so do no elements).
bool lie_alike(Tensor a, Tensor b) {
    if (a.sizes() != b.sizes()) return false;
    for (int64_t k = 0; k < a.dim(); k++)
        if (a.size(k) > 1 && a.stride(k) != b.stride(k) && a.numel()) return false;
    return true;
}
// (gradients, max_norm, out) -> (outputs or None, norm); max_norm None: the norm alone; out None: new tensors
PyObject* clip_gradients(PyObject* const* a) {
    const Reference list{PySequence_Fast(a[0], "gradients: a sequence of tensors is wanted")};
    if (!list.o) throw Raised{};
    const bool writes = a[1] != Py_None;
    const Reference outs{writes && a[2] != Py_None ? PySequence_Fast(a[2], "out: a sequence of tensors is wanted") : nullptr};
    if (writes && a[2] != Py_None && !outs.o) throw Raised{};
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(list.o);
    if (count == 0 || count > INT32_MAX) refuse("gradients: at least one tensor is wanted");
    if (outs.o && PySequence_Fast_GET_SIZE(outs.o) != count) refuse("out: " + std::to_string(count) + " tensors are wanted");
    std::vector<at::Tensor> held;
    std::vector<b200_gradient> gradients(count);
    held.reserve(2 * count);
    for (Py_ssize_t k = 0; k < count; k++) {
        auto name = [&](const char* what) { return std::string(what) + "[" + std::to_string(k) + "]"; };
        PyObject* o = PySequence_Fast_GET_ITEM(list.o, k);
        if (!THPVariable_Check(o)) refuse(name("gradients") + ": a tensor is wanted");
        held.push_back(tensor(o, "gradients"));
        const at::Tensor g = held.back();
        if (!g.is_cuda() || g.device() != held.front().device()) refuse(name("gradients") + ": on another device than the first, or on none");
        if (!among(g.scalar_type(), kFloats)) refuse(name("gradients") + ": this type is not taken here");
        if (!g.is_non_overlapping_and_dense()) refuse(name("gradients") + ": elements must lie side by side");
        gradients[k] = {g.data_ptr(), nullptr, g.numel(), type_of(g.scalar_type())};
    }
    for (Py_ssize_t k = 0; writes && k < count; k++) {
        const at::Tensor g = held[k];
        if (outs.o) {
            held.push_back(tensor(PySequence_Fast_GET_ITEM(outs.o, k), "out"));
            Tensor t = held.back();
            if (t.scalar_type() != g.scalar_type() || !lie_alike(t, g) || t.device() != g.device())
                refuse("out[" + std::to_string(k) + "]: not of its gradient's type, shape, strides and device");
        } else {
            held.push_back(at::detail::empty_strided_cuda(g.sizes(), g.strides(), g.scalar_type(), g.device()));
        }
        gradients[k].out = held.back().data_ptr();
    }
    Tensor first = held.front();
    const at::Tensor norm = empty({}, at::kFloat, first);
    b200_clip_op op{};
    op.count = (int)count, op.gradients = gradients.data(), op.norm = static_cast<float*>(norm.data_ptr());
    const double max_norm = writes ? number(a[1]) : 0;
    if (!(max_norm >= 0)) refuse("max_norm: 0 or above is wanted");
    op.max_norm = (float)max_norm;
    op.max_norm_low = std::isfinite(op.max_norm) ? (float)(max_norm - op.max_norm) : 0.f;
    const at::Tensor scratch = space(b200_op_clip_gradients_workspace, op, first);
    check(b200_op_clip_gradients(device_of(first), stream_of(first), &op));
    // (torch counts what is written in place, so that a backward which has kept such a tensor does not go on with other values; tensors of inference mode have no count)
    for (Py_ssize_t k = 0; outs.o && k < count; k++)
        if (!held[count + k].is_inference()) held[count + k].unsafeGetTensorImpl()->bump_version();
    if (!writes) return Py_BuildValue("(ON)", Py_None, THPVariable_Wrap(norm));
    const Reference clipped{PyList_New(count)};
    if (!clipped.o) throw Raised{};
    for (Py_ssize_t k = 0; k < count; k++) {
        PyObject* o = THPVariable_Wrap(held[count + k]);
        if (!o) throw Raised{};
        PyList_SET_ITEM(clipped.o, k, o);
    }
    return Py_BuildValue("(ON)", clipped.o, THPVariable_Wrap(norm));
}

// (dy, x, x_scale, w, y, y_scale, act, dskip, dw_dtype, need_dx, need_dw, need_dbias) -> (dx, dw, dbias); what is not needed None
PyObject* dense_backward(PyObject* const* a) {
    const at::Tensor dy = tensor(a[0], "dy");
    const auto x = maybe_tensor(a[1], "x"), x_scale = maybe_tensor(a[2], "x's scales"), w = maybe_tensor(a[3], "w"), y = maybe_tensor(a[4], "y"),
               y_scale = maybe_tensor(a[5], "y's scales"), dskip = maybe_tensor(a[7], "dskip");
    const bool need_dx = truth(a[9]), need_dw = truth(a[10]), need_dbias = truth(a[11]);
    b200_dense_grad_op op{};
    op.act = act_of(a[6]);
    op.lddy = matrix(dy, "dy", k16Bits);
    const at::ScalarType kind = dy.scalar_type();
    const int64_t rows = dy.size(0), n_out = dy.size(1);
    if (need_dx && !w) refuse("w: the gradient at the input needs the weights");
    if (need_dw && !x) refuse("x: the gradient at the weights needs the input");
    const int64_t n_in = need_dx ? (w->dim() == 2 ? w->size(0) : 0) : need_dw ? (x->dim() == 2 ? x->size(1) : 0) : 1;
    op.x_type = op.y_type = op.dy_type = type_of(kind);
    auto checkpoint = [&](Tensor t, const std::optional<at::Tensor>& scale, const char* what, const char* whose, int64_t width, int64_t& ld, const void*& at, const float*& scale_at, int32_t& type) {
        ld = matrix(t, what, scale ? at::kFloat8_e4m3fn : kind, rows, width, dy);
        at = t.data_ptr();
        scale_at = vector(scale, whose, rows, dy);
        type = type_of(t.scalar_type());
    };
    if (need_dw) checkpoint(*x, x_scale, "x", "x's scales", n_in, op.ldx, op.x, op.x_scale, op.x_type);
    if (op.act != B200_ACT_NONE) {
        if (!y) refuse("y: the gradient of an activation needs its output");
        checkpoint(*y, y_scale, "y", "y's scales", n_out, op.ldy, op.y, op.y_scale, op.y_type);
    }
    std::optional<at::Tensor> dx, dw, dbias;
    if (need_dx) {
        op.ldw = matrix(*w, "w", kind, n_in, n_out, dy);
        op.w = w->data_ptr();
        if (dskip) op.ldskip = matrix(*dskip, "dskip", kind, rows, n_in, dy), op.dskip = dskip->data_ptr();
        dx = empty({rows, n_in}, kind, dy);
    }
    const at::ScalarType dw_kind = dtype(a[8], "dw_dtype");
    if (dw_kind != at::kFloat && dw_kind != kind) refuse("dw_dtype: this type is not taken here");
    if (need_dw) dw = empty({n_in, n_out}, dw_kind, dy);
    if (need_dbias) dbias = empty({n_out}, at::kFloat, dy);
    op.rows = (int)rows, op.in = (int)n_in, op.out = (int)n_out, op.dw_type = type_of(dw_kind);
    op.lddx = n_in, op.lddw = n_out;
    op.dy = dy.data_ptr(), op.dx = at_of(dx), op.dw = at_of(dw), op.dbias = static_cast<float*>(at_of(dbias));
    const at::Tensor held = space(b200_op_dense_backward_workspace, op, dy);
    check(b200_op_dense_backward(device_of(dy), stream_of(dy), &op));
    return tuple<3>({dx, dw, dbias});
}

template <PyObject* (*Call)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments are wanted, not %zd", N, n);
        return nullptr;
    }
    try {
        return Call(args);
    } catch (const Raised&) {
        return nullptr;
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(memory_error, e.what());
        return nullptr;
    } catch (const std::exception& e) {  // torch's other ones
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
PyObject* set_errors(PyObject*, PyObject* args) {
    PyObject *library, *memory;
    if (!PyArg_ParseTuple(args, "OO", &library, &memory)) return nullptr;
    Py_INCREF(library);
    Py_XSETREF(library_error, library);
    Py_INCREF(memory);
    Py_XSETREF(memory_error, memory);
    Py_RETURN_NONE;
}

#define B200_ENTRY(name, n) {#name, (PyCFunction)(void (*)(void))entry<name, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {B200_ENTRY(rms_norm, 5),
                         B200_ENTRY(rms_norm_backward, 5),
                         B200_ENTRY(pack8, 3),
                         B200_ENTRY(unpack8, 4),
                         B200_ENTRY(dense, 8),
                         B200_ENTRY(dense_backward, 12),
                         B200_ENTRY(pack4, 2),
                         B200_ENTRY(unpack4, 5),
                         B200_ENTRY(dense4, 10),
                         B200_ENTRY(embed, 4),
                         B200_ENTRY(embed_backward, 5),
                         B200_ENTRY(clip_gradients, 3),
                         {"set_errors", set_errors, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls() { return PyModule_Create(&module); }
