// Operator-level entry points of tables whose rows are named by ids: b200_op_embed and its gradient.
#include <algorithm>

#include "kernels_table.cuh"
#include "op_call.h"
#include "with_type.h"

namespace {

using namespace b200;

constexpr int kTableSms = 148;

int check_lists(const char* who, int rows, int slots, int n, int cols, int wide) {
    if (rows < 0 || slots < 1 || n < 1 || cols < 1) return fail(B200_ERR_ARG, "%s: %d lists of %d, %d rows of %d", who, rows, slots, n, cols);
    if ((int64_t)rows * slots > INT32_MAX - 65536) return fail(B200_ERR_UNSUPPORTED, "%s: %d lists of %d are too many", who, rows, slots);
    if (wide != 0 && wide != 1) return fail(B200_ERR_ARG, "%s: wide_ids is %d", who, wide);
    return 0;
}
int check_ids(const char* who, const void* ids, int64_t ld, int rows, int slots, int wide) {
    if (!ids) return fail(B200_ERR_ARG, "%s: ids is NULL", who);
    if ((uintptr_t)ids % (wide ? 8 : 4)) return fail(B200_ERR_ARG, "%s: ids is not aligned to its elements", who);
    if (ld < slots || ld > INT64_MAX / 8 / (rows > 0 ? rows : 1)) return fail(B200_ERR_ARG, "%s: ld of ids is %lld, with lists of %d", who, (long long)ld, slots);
    return 0;
}
bool vectors(const void* at, int64_t ld, int cols, int type) { return cols % 8 == 0 && ((uintptr_t)at | (uintptr_t)(ld * type_bytes(type))) % 16 == 0; }
unsigned ctas_for(int64_t places) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((places + kTableThreads - 1) / kTableThreads, kTableSms * 8)); }

// How ids are sorted: in passes of equal digits, by whole tiles.
struct Sorting {
    int64_t count;
    int passes, bits, tiles;
};
Sorting sorting_of(const b200_embed_grad_op* op) {
    Sorting s{(int64_t)op->rows * op->slots};
    int wanted = 1;
    while (wanted < 31 && op->n >> wanted) wanted++;  // (n itself stands for no row)
    s.passes = (wanted + 7) / 8;
    s.bits = (wanted + s.passes - 1) / s.passes;
    s.tiles = (int)((s.count + kSortTile - 1) / kSortTile);
    return s;
}
// Where the parts of a gradient's workspace begin, in bytes.
struct Space {
    int64_t pairs, more_pairs, counts, start, parts, all;
    int64_t pieces, ldp;
};
Space space_of(const b200_embed_grad_op* op) {
    Space s{};
    if (op->rows == 0) return s;
    auto next = [&](int64_t bytes) {
        const int64_t at = s.all;
        s.all += (bytes + 255) / 256 * 256;
        return at;
    };
    const Sorting sort = sorting_of(op);
    s.pairs = next(sort.count * 8);
    s.more_pairs = next(sort.passes > 1 ? sort.count * 8 : 0);
    s.counts = next(((int64_t)sort.tiles << sort.bits) * 4);
    s.start = next((op->n + 1ll) * 4);
    s.pieces = sort.count > kStretch ? (sort.count + kStretch - 1) / kStretch : 0;  // (shorter lists have no stretch that is cut)
    s.ldp = (op->cols + 7ll) / 8 * 8;
    s.parts = next(2 * s.pieces * s.ldp * 4);
    return s;
}

int check_embed_grad(const b200_embed_grad_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_lists(who, op->rows, op->slots, op->n, op->cols, op->wide_ids)) return rc;
    if (!is_float(op->dy_type) || !is_float(op->dtable_type)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->dy_type, op->dtable_type);
    return 0;
}

}  // namespace

extern "C" {

int b200_op_embed(int device, void* stream, const b200_embed_op* op) {
    const char* who = "op_embed";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_lists(who, op->rows, op->slots, op->n, op->cols, op->wide_ids)) return rc;
    if (!is_float(op->table_type) || !is_float(op->y_type)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->table_type, op->y_type);
    if (op->rows == 0) return 0;
    if (int rc = check_ids(who, op->ids, op->ldids, op->rows, op->slots, op->wide_ids)) return rc;
    if (int rc = check_matrix(who, "table", op->table, op->ldt, op->n, op->cols, op->table_type)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->cols, op->y_type)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    with_float(op->table_type, [&](auto t) {
        with_bool(vectors(op->table, op->ldt, op->cols, op->table_type) && vectors(op->y, op->ldy, op->cols, op->y_type), [&](auto v) {
            embed_kernel<decltype(t), v()><<<ctas_for((int64_t)op->rows * ((op->cols + 7) / 8)), kTableThreads, 0, static_cast<cudaStream_t>(stream)>>>(*op);
        });
    });
    OP_CK(cudaGetLastError());
    return 0;
}

int b200_op_embed_backward_workspace(const b200_embed_grad_op* op, int64_t* bytes) {
    if (int rc = check_embed_grad(op, "op_embed_backward")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_embed_backward: null result");
    *bytes = space_of(op).all;
    return 0;
}

int b200_op_embed_backward(int device, void* stream, const b200_embed_grad_op* op) {
    const char* who = "op_embed_backward";
    if (int rc = check_embed_grad(op, who)) return rc;
    if (int rc = check_matrix(who, "dtable", op->dtable, op->lddt, op->n, op->cols, op->dtable_type)) return rc;
    const Space space = space_of(op);
    if (op->rows) {
        if (int rc = check_ids(who, op->ids, op->ldids, op->rows, op->slots, op->wide_ids)) return rc;
        if (int rc = check_matrix(who, "dy", op->dy, op->lddy, op->rows, op->cols, op->dy_type)) return rc;
        if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, space.all)) return rc;
    }
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (op->rows == 0) {
        OP_CK(cudaMemset2DAsync(op->dtable, op->lddt * type_bytes(op->dtable_type), 0, (size_t)op->cols * type_bytes(op->dtable_type), op->n, s));
        return 0;
    }
    char* base = static_cast<char*>(op->workspace);
    const Sorting sort = sorting_of(op);
    int2* pairs[2] = {reinterpret_cast<int2*>(base + space.pairs), reinterpret_cast<int2*>(base + space.more_pairs)};
    SortPass p{};
    p.ids = op->ids, p.ldids = op->ldids, p.slots = op->slots, p.wide = op->wide_ids, p.n = op->n;
    p.count = sort.count, p.tiles = sort.tiles, p.counts = reinterpret_cast<int*>(base + space.counts), p.bits = sort.bits;
    for (int k = 0; k < sort.passes; k++) {
        p.to = pairs[k & 1];
        p.shift = k * sort.bits;
        OP_CK(launch_step(k > 0, pass_count_kernel, sort.tiles, kSortThreads, 0, s, p));
        OP_CK(launch_step(true, pass_scan_kernel, 1, 1024, 0, s, p.counts, (int64_t)sort.tiles << sort.bits));
        OP_CK(launch_step(true, pass_place_kernel, sort.tiles, kSortThreads, 0, s, p));
        p.from = p.to;
    }
    int* start = reinterpret_cast<int*>(base + space.start);
    OP_CK(launch_step(true, stretches_kernel, (unsigned)((sort.count + kTableThreads) / kTableThreads), kTableThreads, 0, s, p.from, sort.count, op->n, start));
    const TableGrad g{*op, p.from, start, reinterpret_cast<float*>(base + space.parts), space.ldp, space.pieces};
    const bool vec_out = vectors(op->dtable, op->lddt, op->cols, op->dtable_type);
    const int64_t across = (op->cols + 7) / 8;
    cudaError_t rc = cudaSuccess;
    with_float(op->dy_type, [&](auto t) {
        with_bool(vectors(op->dy, op->lddy, op->cols, op->dy_type) && vec_out, [&](auto v) {
            rc = launch_step(true, embed_backward_kernel<decltype(t), v()>, ctas_for((op->n + space.pieces) * across), kTableThreads, 0, s, g);
        });
    });
    OP_CK(rc);
    if (space.pieces) OP_CK(launch_step(true, vec_out ? embed_join_kernel<true> : embed_join_kernel<false>, ctas_for(op->n * across), kTableThreads, 0, s, g));
    return 0;
}

}  // extern "C"
