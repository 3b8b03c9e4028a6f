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

#include <optional>
#include <string>

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
                         {"set_errors", set_errors, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls() { return PyModule_Create(&module); }
