// Operator-level entry points over the rows of a matrix: b200_op_rms_norm and its gradient, b200_op_pack8, b200_op_unpack8.
#include <algorithm>

#include "kernels_rows.cuh"
#include "op_call.h"

namespace {

using namespace b200;

// f(element type) for one of the float types
template <class F>
auto with_float(int type, F f) {
    return type == B200_TYPE_F32 ? f(float{}) : type == B200_TYPE_BF16 ? f(bf16{}) : f(f16{});
}

int row_ctas(int rows) { return std::min(rows, 148 * 8); }
// pieces of the rows for sums over a column
int pieces(int rows, int cols) { return std::max(1, std::min(rows / 16, 148 * 8 / ((cols + kRowThreads - 1) / kRowThreads))); }

int check_norm(const b200_rms_norm_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->cols < 1) return fail(B200_ERR_ARG, "%s: %d rows of %d", who, op->rows, op->cols);
    if (!is_float(op->x_type) || !(is_float(op->y_type) || op->y_type == B200_TYPE_E4M3)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->x_type, op->y_type);
    if (!(op->eps >= 0.f)) return fail(B200_ERR_ARG, "%s: eps must not be negative", who);
    if (op->rows == 0) return 0;
    if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->cols, op->x_type)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->cols, op->y_type)) return rc;
    if (op->residual)
        if (int rc = check_matrix(who, "residual", op->residual, op->ldr, op->rows, op->cols, op->x_type)) return rc;
    if (op->sum)
        if (int rc = check_matrix(who, "sum", op->sum, op->lds, op->rows, op->cols, op->x_type)) return rc;
    if (op->weight)
        if (int rc = check_floats(who, "weight", op->weight)) return rc;
    if (op->rstd)
        if (int rc = check_floats(who, "rstd", op->rstd)) return rc;
    if (op->y_type == B200_TYPE_E4M3)
        if (int rc = check_floats(who, "scale", op->scale)) return rc;
    return 0;
}

int check_norm_grad(const b200_rms_norm_grad_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->cols < 1) return fail(B200_ERR_ARG, "%s: %d rows of %d", who, op->rows, op->cols);
    if (!is_float(op->x_type) || !is_float(op->dy_type)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->x_type, op->dy_type);
    return 0;
}

int64_t norm_grad_workspace(const b200_rms_norm_grad_op* op) {
    return op->dweight && op->rows ? (int64_t)pieces(op->rows, op->cols) * op->cols * 4 : 0;
}

int check_pack(int rows, int cols, int type, const char* who) {
    if (rows < 0 || cols < 1) return fail(B200_ERR_ARG, "%s: %d rows of %d", who, rows, cols);
    if (!is_float(type)) return fail(B200_ERR_UNSUPPORTED, "%s: type %d", who, type);
    return 0;
}

}  // namespace

extern "C" {

int b200_op_rms_norm(int device, void* stream, const b200_rms_norm_op* op) {
    if (int rc = check_norm(op, "op_rms_norm")) return rc;
    if (op->rows == 0) return 0;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_float(op->x_type, [&](auto x) {
        using TX = decltype(x);
        if (op->y_type == B200_TYPE_E4M3)
            rms_norm_kernel<TX, e4m3><<<row_ctas(op->rows), kRowThreads, 0, s>>>(*op);
        else
            with_float(op->y_type, [&](auto y) { rms_norm_kernel<TX, decltype(y)><<<row_ctas(op->rows), kRowThreads, 0, s>>>(*op); });
    });
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_rms_norm_backward_workspace(const b200_rms_norm_grad_op* op, int64_t* bytes) {
    if (int rc = check_norm_grad(op, "op_rms_norm_backward")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_rms_norm_backward: null result");
    *bytes = norm_grad_workspace(op);
    return 0;
}

int b200_op_rms_norm_backward(int device, void* stream, const b200_rms_norm_grad_op* op) {
    const char* who = "op_rms_norm_backward";
    if (int rc = check_norm_grad(op, who)) return rc;
    if (op->dweight)
        if (int rc = check_floats(who, "dweight", op->dweight)) return rc;
    if (op->rows) {
        if (int rc = check_matrix(who, "dy", op->dy, op->lddy, op->rows, op->cols, op->dy_type)) return rc;
        if (int rc = check_matrix(who, "sum", op->sum, op->lds, op->rows, op->cols, op->x_type)) return rc;
        if (int rc = check_floats(who, "rstd", op->rstd)) return rc;
        if (op->weight)
            if (int rc = check_floats(who, "weight", op->weight)) return rc;
        if (op->dsum)
            if (int rc = check_matrix(who, "dsum", op->dsum, op->ldds, op->rows, op->cols, op->x_type)) return rc;
        if (op->dx)
            if (int rc = check_matrix(who, "dx", op->dx, op->lddx, op->rows, op->cols, op->x_type)) return rc;
        if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, norm_grad_workspace(op))) return rc;
    }
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (op->rows == 0) {
        if (op->dweight) OP_CK(cudaMemsetAsync(op->dweight, 0, (size_t)op->cols * 4, s));
        return 0;
    }
    const int column_ctas = (op->cols + kRowThreads - 1) / kRowThreads, n = pieces(op->rows, op->cols);
    float* parts = static_cast<float*>(op->workspace);
    with_float(op->x_type, [&](auto x) {
        with_float(op->dy_type, [&](auto dy) {
            if (op->dx) rms_norm_dx_kernel<decltype(x), decltype(dy)><<<row_ctas(op->rows), kRowThreads, 0, s>>>(*op);
            if (op->dweight) rms_norm_dweight_kernel<decltype(x), decltype(dy)><<<dim3(column_ctas, n), kRowThreads, 0, s>>>(*op, parts);
        });
    });
    if (op->dweight) add_parts_kernel<<<column_ctas, kRowThreads, 0, s>>>(parts, n, op->cols, op->dweight);
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_pack8(int device, void* stream, const b200_pack8_op* op) {
    const char* who = "op_pack8";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_pack(op->rows, op->cols, op->x_type, who)) return rc;
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    if (op->rows || op->by_column)
        if (int rc = check_floats(who, "scale", op->scale)) return rc;
    if (op->rows) {
        if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->cols, op->x_type)) return rc;
        if (int rc = check_matrix(who, "q", op->q, op->ldq, op->rows, op->cols, B200_TYPE_E4M3)) return rc;
    } else if (!op->by_column) {
        return 0;
    }
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!op->by_column) {
        with_float(op->x_type, [&](auto x) { pack8_rows_kernel<decltype(x)><<<row_ctas(op->rows), kRowThreads, 0, s>>>(*op); });
    } else {
        const dim3 grid((op->cols + kRowThreads - 1) / kRowThreads, pieces(op->rows, op->cols));
        OP_CK(cudaMemsetAsync(op->scale, 0, (size_t)op->cols * 4, s));
        with_float(op->x_type, [&](auto x) {
            column_scales_kernel<decltype(x)><<<grid, kRowThreads, 0, s>>>(*op);
            pack8_columns_kernel<decltype(x)><<<grid, kRowThreads, 0, s>>>(*op);
        });
    }
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_unpack8(int device, void* stream, const b200_unpack8_op* op) {
    const char* who = "op_unpack8";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_pack(op->rows, op->cols, op->y_type, who)) return rc;
    if (op->rows == 0) return 0;
    if (int rc = check_matrix(who, "q", op->q, op->ldq, op->rows, op->cols, B200_TYPE_E4M3)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->cols, op->y_type)) return rc;
    if (int rc = check_floats(who, "scale", op->scale)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    with_float(op->y_type, [&](auto y) { unpack8_kernel<decltype(y)><<<row_ctas(op->rows), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(*op); });
    OP_CK(cudaGetLastError());
    return 0;
}

}  // extern "C"
