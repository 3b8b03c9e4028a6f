// Operator-level entry points over the rows of a matrix: b200_op_rms_norm and its gradient, b200_op_pack8, b200_op_unpack8.
#include <algorithm>

#include "kernels_rows.cuh"
#include "op_call.h"
#include "with_type.h"

namespace {

using namespace b200;

// How a launch deals rows out: `warps` of a CTA to a row (1: every warp one of its own), `vectors` of eight elements a lane.
struct RowShape {
    int warps, vectors, threads;
    int64_t groups;  // rows of a CTA
};
// A lane takes `best` vectors where the row has them, so that a warp has 4 KB on their way and registers for many warps; wider rows have
// more warps, up to kRowWarpsMost, then more vectors.  With fewer rows than the GPU has warps to spare (kFewRows) a row is shared out, a vector a lane.
// Measured, us: norm with residual to 8 bits, 131072 x 2048 bf16, of 8 / 4 / 2 vectors 328 / 290 / 349; fp32 without residual 300 / 278 /
// 259; gradient of 131072 x 2048 bf16 rows, of 4 / 2 / 1 505 / 405 / 614.  Norm to 8 bits of 592 rows of 2048 shared out 3.5, as above 4.5; of
// 1000 rows 5.3 and 4.9, of 2300 rows 9.1 and 8.3; of rows of 520 3.0 and 3.7, 3.3 and 3.9, 4.5 and 4.4.
constexpr int kFewRows = 148 * 4;
RowShape row_shape(int64_t rows, int cols, int best, bool several) {
    RowShape s;
    const int needed = (cols + 255) / 256;  // vectors of one warp's lanes
    s.warps = std::max(1, std::min(kRowWarpsMost, rows <= kFewRows ? needed : (needed + best - 1) / best));
    s.vectors = (needed + s.warps - 1) / s.warps;
    s.groups = several && rows > kFewRows ? kRowWarpsMost / s.warps : s.warps == 1 ? 4 : 1;
    s.threads = 32 * s.warps * (int)s.groups;
    return s;
}
RowShape pack_shape(int64_t rows, int cols) { return row_shape(rows, cols, 8, false); }
RowShape norm_shape(int64_t rows, int cols, int type) { return row_shape(rows, cols, type == B200_TYPE_F32 ? 2 : 4, false); }
RowShape grad_shape(int64_t rows, int cols) { return row_shape(rows, cols, 2, true); }  // (fewer sums to leave behind)
// f(std::integral_constant) for the smallest of 1, 2, 4, ... that holds `vectors`
template <int Most, class F>
void with_vectors(int vectors, F f) {
    if (vectors <= 1)
        f(std::integral_constant<int, 1>{});
    else if (vectors <= 2)
        f(std::integral_constant<int, 2>{});
    else if (vectors <= 4 || Most == 4)
        f(std::integral_constant<int, 4>{});
    else
        f(std::integral_constant<int, Most == 4 ? 4 : 8>{});
}
constexpr int kRowVectors = 8, kGradVectors = 4;  // most of a lane
constexpr int kRowCols = 256 * kRowWarpsMost * kRowVectors, kGradCols = 256 * kRowWarpsMost * kGradVectors;
int any_ctas(int rows) { return std::min(rows, 148 * 8); }
// pieces of the rows for sums over a column by CTAs that take `width` columns and, of those, `at_once` rows
int pieces(int64_t rows, int cols, int width, int at_once) {
    const int64_t across = (cols + width - 1) / width;
    return (int)std::max<int64_t>(1, std::min<int64_t>({rows / (4 * at_once), 148 * 8 / across, 65535}));
}
// threads side by side in a row of `vectors`
int threads_across(int vectors) {
    int t = 1;
    while (t < kRowThreads && t < vectors) t *= 2;
    return t;
}
bool aligned(const void* at, int64_t ld, int type, int to) { return ((uintptr_t)at | (uintptr_t)(ld * type_bytes(type))) % to == 0; }
bool aligned8(const void* at, int64_t ld, int type) { return aligned(at, ld, type, 8 * type_bytes(type)); }  // vectors of eight elements

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

// CTAs of the gradient per SM, each of which leaves a row of sums: as many as run at once.  Of 1 / 2 / 3 / 4, us: 5003 x 520 bf16 13.6 / 10.7 /
// 14.3 / 12.9, 5003 x 1024 14.1 / 11.8 / 15.7 / 14.5, 131072 x 1024 fp32 344 / 231 / 282 / 234, 131072 x 2048 bf16 470 / 310 / 390 / 314.
constexpr int kGradCtas = 2;
int norm_grad_ctas(const b200_rms_norm_grad_op* op) {
    if (op->cols > kGradCols) return pieces(op->rows, op->cols, kRowThreads, 4);
    const RowShape g = grad_shape(op->rows, op->cols);
    return (int)std::min<int64_t>((op->rows + g.groups - 1) / g.groups, 148 * kGradCtas);
}
int64_t norm_grad_workspace(const b200_rms_norm_grad_op* op) { return op->dweight && op->rows ? (int64_t)norm_grad_ctas(op) * op->cols * 4 : 0; }

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
    if (op->cols > kRowCols) {
        with_float(op->x_type, [&](auto x) { rms_norm_any_kernel<decltype(x)><<<any_ctas(op->rows), kRowThreads, 0, s>>>(*op); });
    } else {
        const bool vec = op->cols % 8 == 0 && aligned8(op->x, op->ldx, op->x_type) && aligned8(op->y, op->ldy, op->y_type) && (!op->residual || aligned8(op->residual, op->ldr, op->x_type)) &&
                         (!op->sum || aligned8(op->sum, op->lds, op->x_type)) && (uintptr_t)op->weight % 32 == 0;
        const RowShape g = norm_shape(op->rows, op->cols, op->x_type);
        with_float(op->x_type, [&](auto x) {
            with_bool(vec, [&](auto v) {
                with_vectors<kRowVectors>(g.vectors, [&](auto nv) {
                    auto go = [&](auto kernel) { kernel<<<(unsigned)((op->rows + g.groups - 1) / g.groups), g.threads, 0, s>>>(*op, g.warps, 1.0 / op->cols); };
                    if (op->y_type == B200_TYPE_E4M3)
                        go(rms_norm_kernel<decltype(x), nv(), v(), true>);
                    else
                        go(rms_norm_kernel<decltype(x), nv(), v(), false>);
                });
            });
        });
    }
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
    const int ctas = norm_grad_ctas(op);
    float* parts = static_cast<float*>(op->workspace);
    if (op->cols > kGradCols) {
        with_float(op->x_type, [&](auto x) {
            with_float(op->dy_type, [&](auto dy) {
                if (op->dx) rms_norm_dx_any_kernel<decltype(x), decltype(dy)><<<any_ctas(op->rows), kRowThreads, 0, s>>>(*op);
                if (op->dweight)
                    rms_norm_dweight_any_kernel<decltype(x), decltype(dy)><<<dim3((op->cols + kRowThreads - 1) / kRowThreads, ctas), kRowThreads, 0, s>>>(*op, parts);
            });
        });
    } else if (op->dx || op->dweight) {
        const bool vec = op->cols % 8 == 0 && aligned8(op->dy, op->lddy, op->dy_type) && aligned8(op->sum, op->lds, op->x_type) && (!op->dx || aligned8(op->dx, op->lddx, op->x_type)) &&
                         (!op->dsum || aligned8(op->dsum, op->ldds, op->x_type)) && (uintptr_t)op->weight % 32 == 0;
        const RowShape g = grad_shape(op->rows, op->cols);
        const size_t shared = op->dweight && g.groups > 1 ? (size_t)g.groups * op->cols * 4 : 0;  // at most 4 x 1024 floats
        with_float(op->x_type, [&](auto x) {
            with_float(op->dy_type, [&](auto dy) {
                with_bool(vec, [&](auto v) {
                    with_vectors<kGradVectors>(g.vectors, [&](auto nv) {
                        rms_norm_backward_kernel<decltype(x), decltype(dy), nv(), v()><<<ctas, g.threads, shared, s>>>(*op, parts, g.warps);
                    });
                });
            });
        });
    }
    OP_CK(cudaGetLastError());
    if (op->dweight) OP_CK(launch_step(true, add_parts_kernel, (op->cols + 31) / 32, kAddThreads, 0, s, parts, ctas, op->cols, op->dweight));
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
    const bool vec = op->cols % 8 == 0 && aligned8(op->x, op->ldx, op->x_type) && aligned8(op->q, op->ldq, B200_TYPE_E4M3);
    if (op->by_column) {
        const int across = threads_across(vec ? op->cols / 8 : op->cols), width = across * (vec ? 8 : 1);
        const dim3 grid((op->cols + width - 1) / width, pieces(op->rows, op->cols, width, kRowThreads / across));
        // (every piece sends each column's magnitude to one address: four CTAs per SM at most)
        const dim3 scales_grid(grid.x, std::max(1u, std::min(grid.y, 592u / grid.x)));
        OP_CK(cudaMemsetAsync(op->scale, 0, (size_t)op->cols * 4, s));
        with_float(op->x_type, [&](auto x) {
            with_bool(vec, [&](auto v) {
                column_scales_kernel<decltype(x), v() ? 8 : 1><<<scales_grid, kRowThreads, 0, s>>>(*op, across);
                pack8_columns_kernel<decltype(x), v() ? 8 : 1><<<grid, kRowThreads, 0, s>>>(*op, across);
            });
        });
    } else if (op->cols > kRowCols) {
        with_float(op->x_type, [&](auto x) { pack8_rows_any_kernel<decltype(x)><<<any_ctas(op->rows), kRowThreads, 0, s>>>(*op); });
    } else {
        const RowShape g = pack_shape(op->rows, op->cols);
        with_float(op->x_type, [&](auto x) {
            with_bool(vec, [&](auto v) {
                with_vectors<kRowVectors>(g.vectors, [&](auto nv) {
                    auto go = [&](auto kernel) { kernel<<<(unsigned)((op->rows + g.groups - 1) / g.groups), g.threads, 0, s>>>(*op, g.warps); };
                    if (op->act == B200_ACT_NONE)
                        go(pack8_rows_kernel<decltype(x), nv(), v(), false>);
                    else
                        go(pack8_rows_kernel<decltype(x), nv(), v(), true>);
                });
            });
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
    const bool on16 = aligned8(op->y, op->ldy, op->y_type);
    const int v = on16 && op->cols % 16 == 0 && aligned(op->q, op->ldq, B200_TYPE_E4M3, 16) ? 16 : on16 && op->cols % 8 == 0 && aligned(op->q, op->ldq, B200_TYPE_E4M3, 8) ? 8 : 1;
    const int across = threads_across(op->cols / v), rows = kRowThreads / across * kUnpackRows;
    const unsigned ctas = (unsigned)(((int64_t)op->rows + rows - 1) / rows);
    with_float(op->y_type, [&](auto y) {
        using TY = decltype(y);
        auto go = [&](auto kernel) { kernel<<<ctas, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(*op, across); };
        v == 16 ? go(unpack8_kernel<TY, 16>) : v == 8 ? go(unpack8_kernel<TY, 8>) : go(unpack8_kernel<TY, 1>);
    });
    OP_CK(cudaGetLastError());
    return 0;
}

}  // extern "C"
