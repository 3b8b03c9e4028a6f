// Operator-level entry points of dense layers: b200_op_dense and its gradient.
#include <algorithm>

#include "kernels_product.cuh"
#include "kernels_rows.cuh"
#include "op_call.h"

namespace {

using namespace b200;

int launch_product(const Product& p, cudaStream_t s) {
    if ((p.m + 63) / 64 > 65535) return fail(B200_ERR_UNSUPPORTED, "too many rows");
    product_kernel<<<dim3((unsigned)((p.n + 63) / 64), (unsigned)((p.m + 63) / 64)), 256, 0, s>>>(p);
    OP_CK(cudaGetLastError());
    return 0;
}

int pieces(int rows, int cols) { return std::max(1, std::min(rows / 16, 148 * 8 / ((cols + 255) / 256))); }

int check_dense(const b200_dense_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->in < 1 || op->out < 1) return fail(B200_ERR_ARG, "%s: %d rows, %d in, %d out", who, op->rows, op->in, op->out);
    if (!(is_16_bits(op->x_type) || op->x_type == B200_TYPE_E4M3) || !is_float(op->y_type))
        return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->x_type, op->y_type);
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    return 0;
}

int check_dense_grad(const b200_dense_grad_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->rows < 0 || op->in < 1 || op->out < 1) return fail(B200_ERR_ARG, "%s: %d rows, %d in, %d out", who, op->rows, op->in, op->out);
    auto checkpoint = [&](int type) { return type == op->dy_type || (type == B200_TYPE_E4M3 && op->dy_type == B200_TYPE_BF16); };
    if (!is_16_bits(op->dy_type) || !checkpoint(op->x_type) || !checkpoint(op->y_type) || !(op->dw_type == B200_TYPE_F32 || op->dw_type == op->dy_type))
        return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d, %d, %d", who, op->dy_type, op->x_type, op->y_type, op->dw_type);
    if (!is_act(op->act)) return fail(B200_ERR_ARG, "%s: %d names no activation", who, op->act);
    return 0;
}

// Where the parts of a workspace begin, in bytes.
struct GradSpace {
    int64_t dz, parts, all;
};
GradSpace grad_space(const b200_dense_grad_op* op) {
    GradSpace s{};
    if (op->rows == 0) return s;
    auto next = [&](int64_t bytes) {
        const int64_t at = s.all;
        s.all += (bytes + 255) / 256 * 256;
        return at;
    };
    s.dz = next(op->act != B200_ACT_NONE && (op->dx || op->dw) ? (int64_t)op->rows * op->out * 2 : 0);
    s.parts = next(op->dbias ? (int64_t)pieces(op->rows, op->out) * op->out * 4 : 0);
    return s;
}

}  // namespace

extern "C" {

int b200_op_dense_workspace(const b200_dense_op* op, int64_t* bytes) {
    if (int rc = check_dense(op, "op_dense")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_dense: null result");
    *bytes = 0;
    return 0;
}

int b200_op_dense(int device, void* stream, const b200_dense_op* op) {
    const char* who = "op_dense";
    if (int rc = check_dense(op, who)) return rc;
    if (op->rows == 0) return 0;
    const bool packed = op->x_type == B200_TYPE_E4M3;
    if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->in, op->x_type)) return rc;
    if (int rc = check_matrix(who, "w", op->w, op->ldw, op->in, op->out, op->x_type)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->out, op->y_type)) return rc;
    if (op->residual)
        if (int rc = check_matrix(who, "residual", op->residual, op->ldr, op->rows, op->out, op->y_type)) return rc;
    if (op->bias)
        if (int rc = check_floats(who, "bias", op->bias)) return rc;
    if (packed) {
        if (int rc = check_floats(who, "x_scale", op->x_scale)) return rc;
        if (int rc = check_floats(who, "w_scale", op->w_scale)) return rc;
    }
    OnDevice on(device);
    OP_CK(on.status);
    Product p{};
    p.m = op->rows, p.n = op->out, p.k = op->in;
    p.a = op->x, p.a_m = op->ldx, p.a_k = 1, p.a_type = op->x_type;
    p.b = op->w, p.b_k = op->ldw, p.b_n = 1, p.b_type = op->x_type;
    if (packed) p.a_scale_m = op->x_scale, p.b_scale_n = op->w_scale;
    p.bias = op->bias, p.residual = op->residual, p.ldr = op->ldr;
    p.d = op->y, p.ldd = op->ldy, p.d_type = op->y_type, p.act = op->act;
    return launch_product(p, static_cast<cudaStream_t>(stream));
}

int b200_op_dense_backward_workspace(const b200_dense_grad_op* op, int64_t* bytes) {
    if (int rc = check_dense_grad(op, "op_dense_backward")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_dense_backward: null result");
    *bytes = grad_space(op).all;
    return 0;
}

int b200_op_dense_backward(int device, void* stream, const b200_dense_grad_op* op) {
    const char* who = "op_dense_backward";
    if (int rc = check_dense_grad(op, who)) return rc;
    const bool acts = op->act != B200_ACT_NONE;
    if (op->dw)
        if (int rc = check_matrix(who, "dw", op->dw, op->lddw, op->in, op->out, op->dw_type)) return rc;
    if (op->dbias)
        if (int rc = check_floats(who, "dbias", op->dbias)) return rc;
    const GradSpace space = grad_space(op);
    if (op->rows) {
        if (int rc = check_matrix(who, "dy", op->dy, op->lddy, op->rows, op->out, op->dy_type)) return rc;
        if (acts) {
            if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->out, op->y_type)) return rc;
            if (op->y_type == B200_TYPE_E4M3)
                if (int rc = check_floats(who, "y_scale", op->y_scale)) return rc;
        }
        if (op->dw) {
            if (int rc = check_matrix(who, "x", op->x, op->ldx, op->rows, op->in, op->x_type)) return rc;
            if (op->x_type == B200_TYPE_E4M3)
                if (int rc = check_floats(who, "x_scale", op->x_scale)) return rc;
        }
        if (op->dx) {
            if (int rc = check_matrix(who, "dx", op->dx, op->lddx, op->rows, op->in, op->dy_type)) return rc;
            if (int rc = check_matrix(who, "w", op->w, op->ldw, op->in, op->out, op->dy_type)) return rc;
            if (op->dskip)
                if (int rc = check_matrix(who, "dskip", op->dskip, op->ldskip, op->rows, op->in, op->dy_type)) return rc;
        }
        if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, space.all)) return rc;
    }
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (op->rows == 0) {
        if (op->dw) OP_CK(cudaMemset2DAsync(op->dw, op->lddw * type_bytes(op->dw_type), 0, (size_t)op->out * type_bytes(op->dw_type), op->in, s));
        if (op->dbias) OP_CK(cudaMemsetAsync(op->dbias, 0, (size_t)op->out * 4, s));
        return 0;
    }
    char* base = static_cast<char*>(op->workspace);
    const bool products = op->dx || op->dw;
    void* dz = acts && products ? base + space.dz : nullptr;
    float* parts = op->dbias ? reinterpret_cast<float*>(base + space.parts) : nullptr;
    if (dz || parts) {
        const int n = pieces(op->rows, op->out), ctas = (op->out + 255) / 256;
        dense_dz_kernel<<<dim3(ctas, n), 256, 0, s>>>(*op, dz, parts);
        if (parts) add_parts_kernel<<<ctas, kRowThreads, 0, s>>>(parts, n, op->out, op->dbias);
    }
    OP_CK(cudaGetLastError());
    const void* g = dz ? dz : op->dy;
    const int64_t ldg = dz ? op->out : op->lddy;
    if (op->dx) {
        Product p{};
        p.m = op->rows, p.n = op->in, p.k = op->out;
        p.a = g, p.a_m = ldg, p.a_k = 1, p.a_type = op->dy_type;
        p.b = op->w, p.b_k = 1, p.b_n = op->ldw, p.b_type = op->dy_type;
        p.residual = op->dskip, p.ldr = op->ldskip;
        p.d = op->dx, p.ldd = op->lddx, p.d_type = op->dy_type;
        if (int rc = launch_product(p, s)) return rc;
    }
    if (op->dw) {
        Product p{};
        p.m = op->in, p.n = op->out, p.k = op->rows;
        p.a = op->x, p.a_m = 1, p.a_k = op->ldx, p.a_type = op->x_type, p.a_scale_k = op->x_type == B200_TYPE_E4M3 ? op->x_scale : nullptr;
        p.b = g, p.b_k = ldg, p.b_n = 1, p.b_type = op->dy_type;
        p.d = op->dw, p.ldd = op->lddw, p.d_type = op->dw_type;
        if (int rc = launch_product(p, s)) return rc;
    }
    return 0;
}

}  // extern "C"
