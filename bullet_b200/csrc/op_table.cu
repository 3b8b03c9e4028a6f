// Operator-level entry points of tables whose rows are named by ids: b200_op_embed and its gradient.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kernels_table.cuh"
#include "op_call.h"
#include "with_type.h"

namespace {

using namespace b200;

constexpr int kTableSms = 148;
constexpr int kFewLists = 16, kFewMost = 512;  // of a warp (5003 lists of 520 bf16 columns, 8 rows: at least 64 13 us, 32 9.0, 16 7.5)

int check_lists(const char* who, int rows, int slots, int n, int cols, int wide, float scale) {
    if (rows < 0 || slots < 1 || n < 1 || cols < 1) return fail(B200_ERR_ARG, "%s: %d lists of %d, %d rows of %d", who, rows, slots, n, cols);
    if ((int64_t)rows * slots > INT32_MAX - 65536) return fail(B200_ERR_UNSUPPORTED, "%s: %d lists of %d are too many", who, rows, slots);
    if (wide != 0 && wide != 1) return fail(B200_ERR_ARG, "%s: wide_ids is %d", who, wide);
    if (!std::isfinite(scale)) return fail(B200_ERR_ARG, "%s: scale is not finite", who);
    return 0;
}
int check_ids(const char* who, const void* ids, int64_t ld, int rows, int slots, int wide) {
    if (!ids) return fail(B200_ERR_ARG, "%s: ids is NULL", who);
    if ((uintptr_t)ids % (wide ? 8 : 4)) return fail(B200_ERR_ARG, "%s: ids is not aligned to its elements", who);
    if (ld < slots || ld > INT64_MAX / 8 / (rows > 0 ? rows : 1)) return fail(B200_ERR_ARG, "%s: ld of ids is %lld, with lists of %d", who, (long long)ld, slots);
    return 0;
}
// How many bytes of a row of `type` a lane takes: 32 or 16 where rows start on 16, fewer where the warp would have lanes to spare, 0 (single elements) where rows start anywhere.
// (Us, 131072 lists of 32 ids, bf16, and their gradient by 12288 rows: rows of 64 columns by 16 bytes 156 and 390, by 8 128 and 376, by 4 122 and 354; of 128 columns 159 and
// 393, 125 and 367, 237 and 538; of 256 columns 164 and 438, 246 and 626.)
int bytes_of(const void* at, int64_t ld, int cols, int type, int most) {
    const int64_t size = type_bytes(type), row = cols * size;
    const auto on = [&](int bytes) { return ((uintptr_t)at | (uintptr_t)(ld * size) | (uintptr_t)row) % bytes == 0; };
    if (row > 256 && on(16)) return most == 32 && (row + 1023) / 1024 * 1024 - row <= row / 8 ? 32 : 16;  // (an eighth of the lanes to spare at most)
    if (row > 512) return 0;
    if (row > 128 && on(8)) return 8;
    return on(4) ? 4 : 0;
}
// How many warps' columns a row has.
int across_of(int bytes, int cols, int type) { return (cols - 1) / (32 * (bytes ? bytes : 16) / type_bytes(type)) + 1; }
// What warps there are for `rows` of them, and the bytes of their lanes: 16 at most, and as many rows on their way as registers hold, where that makes few warps.
struct Lines {
    int bytes, across;
    int64_t warps;
    bool few;
};
Lines lines_of(const void* at, int64_t ld, int cols, int type, int64_t rows, int few_warps) {
    Lines l;
    l.bytes = bytes_of(at, ld, cols, type, 32);
    l.few = l.bytes && rows * across_of(l.bytes, cols, type) <= few_warps;
    if (l.few) l.bytes = std::min(l.bytes, 16);
    l.across = across_of(l.bytes, cols, type);
    l.warps = rows * l.across;
    return l;
}
// Whether rows of `type` take `each` elements together.
bool together(const void* at, int64_t ld, int type, int each) {
    const int64_t bytes = std::min(16, each * type_bytes(type));
    return ((uintptr_t)at | (uintptr_t)(ld * type_bytes(type))) % bytes == 0;
}
template <class F>
void with_bytes(int bytes, F f) {
    if (bytes == 32)
        f(std::integral_constant<int, 32>{});
    else if (bytes == 16)
        f(std::integral_constant<int, 16>{});
    else if (bytes == 8)
        f(std::integral_constant<int, 8>{});
    else if (bytes == 4)
        f(std::integral_constant<int, 4>{});
    else
        f(std::integral_constant<int, 0>{});
}
// (More than run at once, as stretches are of all lengths: by 8 an SM the features' gradient takes 81.6 us and one of 131072 ids of 12288 rows 84.8, by 12 80.5 and
// 81.5, by 48 83.4 and 78.3, but lookups longer.)
unsigned ctas_for(int64_t warps) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((warps + kTableThreads / 32 - 1) / (kTableThreads / 32), kTableSms * 12)); }

// How ids are sorted: in passes of equal digits, by whole tiles, or by one CTA.
struct Sorting {
    int64_t count;
    int passes, bits, tiles;
    bool one() const { return count <= kSortOne; }
    bool places;  // no starts: the table has more rows than there are ids
};
Sorting sorting_of(const b200_embed_grad_op* op) {
    Sorting s{(int64_t)op->rows * op->slots};
    int wanted = 1;
    while (wanted < 31 && (op->n - 1) >> wanted) wanted++;
    s.passes = (wanted + 7) / 8;
    s.bits = (wanted + s.passes - 1) / s.passes;
    s.tiles = (int)((s.count + kSortTile - 1) / kSortTile);
    // (us without starts and with them, bf16: 65536 ids of 128 columns, 32768 rows of the table 43 and 35, 131072 58 and 60, 262144 66 and 81; 8192 ids, 8192 rows 37 and 39,
    // 2^20 76 and 584)
    s.places = op->n > s.count;
    return s;
}
// Where the parts of a gradient's workspace begin, in bytes.
struct Space {
    int64_t pairs, more_pairs, counts, start, numbers, done, pieces, parts, all;
    int64_t ldp;
    int piece;
    Lines lines;
    bool cuts;
};
// Tables of few rows: how lists are cut up.  (Us, bf16, 8 rows of 1024 columns, with ids sorted and so: 1024 lists 17 and 8, 131072 86 and 56, 262144 165 and 105.)
bool few_rows(const b200_embed_grad_op* op) { return op->n <= kFewRows && op->slots == 1; }
struct Few {
    int bytes, lists, chunks, across, shared;  // of a lane, as bytes_of; lists of a warp; bytes of a CTA's sums
};
Few few_of(const b200_embed_grad_op* op) {
    Few f;
    f.bytes = bytes_of(op->dy, op->lddy, op->cols, op->dy_type, 16);
    if (f.bytes == 16 && type_bytes(op->dy_type) == 2 && op->n > 13) f.bytes = 8;  // (or an SM has room for one CTA's sums: 262144 x 1024, 16 rows 152 us instead of 210)
    f.across = across_of(f.bytes, op->cols, op->dy_type);
    f.shared = kFewWarps * op->n * 32 * (f.bytes ? f.bytes : 16) / type_bytes(op->dy_type) * 4;
    // As many CTAs as run at once, or a multiple of that where warps would add up more than kFewMost lists.  (262144 x 1024 fp32: by kFewMost alone 250 us, 180.)
    const int64_t at_once = (int64_t)kTableSms * std::max(1, std::min(3, 230000 / (f.shared + 1024))), chunks = std::max<int64_t>(1, at_once / f.across);
    const auto over = [](int64_t all, int64_t each) { return (all + each - 1) / each; };
    const int64_t times = over(over(op->rows, chunks * kFewWarps), kFewMost);
    f.lists = (int)std::max<int64_t>(kFewLists, over(op->rows, chunks * times * kFewWarps));
    f.chunks = (int)over(op->rows, (int64_t)f.lists * kFewWarps);
    return f;
}
Space space_of(const b200_embed_grad_op* op) {
    Space s{};
    if (op->rows == 0) return s;
    if (few_rows(op)) {
        const Few f = few_of(op);
        if (f.chunks > 1) s.all = (int64_t)f.chunks * f.across * f.shared / kFewWarps;
        return s;
    }
    auto next = [&](int64_t bytes) {
        const int64_t at = s.all;
        s.all += (bytes + 255) / 256 * 256;
        return at;
    };
    const Sorting sort = sorting_of(op);
    s.pairs = next(sort.count * 8);
    if (!sort.one()) {
        s.more_pairs = next(sort.passes > 1 ? sort.count * 8 : 0);
        s.counts = next((((int64_t)sort.tiles + 1) << sort.bits) * 4);
    }
    if (!sort.places) s.start = next((op->n + 1ll) * 4);
    s.numbers = next(16);
    // Pieces of 16 for few ids, whose longest stretches then have warps enough (before tables of few rows had kernels of their own: 5003 ids of 8 rows of 520, 64 27 us,
    // 16 23), of 64 for many, as each piece costs its part of the joining (131072 ids of 8 rows of 1024: 16 159 us, 32 118, 64 90; 2^20 lists' ids of 768 rows of 256: 64 100,
    // 512 128); more where they would take more room.
    s.piece = 16;
    while (s.piece < 64 ? sort.count / s.piece > 2048 : s.piece < 512 && sort.count / s.piece > 16384) s.piece *= 2;
    s.cuts = sort.count > kLongest;
    s.lines = lines_of(op->dy, op->lddy, op->cols, op->dy_type, (sort.places ? sort.count : op->n) + (s.cuts ? sort.count / s.piece : 0), kTableSms * 16);
    if (s.cuts) {  // (whole pieces, and of each long stretch one that is none)
        const int64_t pieces = sort.count / s.piece + std::min<int64_t>(op->n, sort.count / kLongest);
        s.done = next(pieces * s.lines.across * 4);
        s.pieces = next(pieces * (int64_t)sizeof(Piece8));
        s.ldp = (op->cols + 7ll) / 8 * 8;
        s.parts = next(pieces * s.ldp * 4);
    }
    return s;
}

template <class T, int BYTES>
int few_rows_gradient(const b200_embed_grad_op* op, const Few& few, cudaStream_t s) {
    FewRows f{*op, static_cast<float*>(op->workspace), few.lists, few.chunks, few.across};
    static std::atomic<uint64_t> allowed;  // a bit per device
    int device = 0;
    OP_CK(cudaGetDevice(&device));
    if (device >= 64 || !(allowed >> device & 1)) {
        OP_CK(cudaFuncSetAttribute(few_rows_kernel<T, BYTES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewWarps * kFewRows * FewSums<T, BYTES>::kRow * 4));
        if (device < 64) allowed |= (uint64_t)1 << device;
    }
    OP_CK(launch_step(false, few_rows_kernel<T, BYTES>, (unsigned)(few.chunks * few.across), kTableThreads, (size_t)few.shared, s, f));
    if (few.chunks > 1) OP_CK(launch_step(true, few_join_kernel<T, BYTES>, (unsigned)(few.across * op->n * FewSums<T, BYTES>::kMany), kTableThreads, 0, s, f));
    return 0;
}

// The whole gradient 0.
int zeros(const b200_embed_grad_op* op, cudaStream_t s) {
    const int64_t row = (int64_t)op->cols * type_bytes(op->dtable_type), apart = op->lddt * type_bytes(op->dtable_type);
    if (apart == row || op->n == 1) {
        OP_CK(cudaMemsetAsync(op->dtable, 0, (size_t)(row * op->n), s));
    } else if (apart <= INT32_MAX) {
        OP_CK(cudaMemset2DAsync(op->dtable, (size_t)apart, 0, (size_t)row, (size_t)op->n, s));
    } else {  // (further apart than that call takes, and so few)
        for (int64_t t = 0; t < op->n; t++) OP_CK(cudaMemsetAsync(static_cast<char*>(op->dtable) + t * apart, 0, (size_t)row, s));
    }
    return 0;
}

int check_embed_grad(const b200_embed_grad_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_lists(who, op->rows, op->slots, op->n, op->cols, op->wide_ids, op->scale)) return rc;
    if (!is_float(op->dy_type) || !is_float(op->dtable_type)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->dy_type, op->dtable_type);
    return 0;
}

}  // namespace

extern "C" {

int b200_op_embed(int device, void* stream, const b200_embed_op* op) {
    const char* who = "op_embed";
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (int rc = check_lists(who, op->rows, op->slots, op->n, op->cols, op->wide_ids, op->scale)) return rc;
    if (!is_float(op->table_type) || !is_float(op->y_type)) return fail(B200_ERR_UNSUPPORTED, "%s: types %d, %d", who, op->table_type, op->y_type);
    if (op->rows == 0) return 0;
    if (int rc = check_ids(who, op->ids, op->ldids, op->rows, op->slots, op->wide_ids)) return rc;
    if (int rc = check_matrix(who, "table", op->table, op->ldt, op->n, op->cols, op->table_type)) return rc;
    if (int rc = check_matrix(who, "y", op->y, op->ldy, op->rows, op->cols, op->y_type)) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const Lines lines = lines_of(op->table, op->ldt, op->cols, op->table_type, op->rows, kTableSms * 8);
    // Short lists: as many of a warp as leave an SM 32 warps, up to all that its lanes have indices of.  (5003 lists of one id, 1024 columns: 32 of a warp 14 us, four 5.3.)
    const int at_once = std::max(1, kEmbedAhead / op->slots), most = 32 / std::min(32, op->slots) / at_once * at_once;
    const int lists = (int)std::min<int64_t>(most, (lines.warps / (kTableSms * 32) + at_once) / at_once * at_once);
    with_float(op->table_type, [&](auto t) {
        with_bytes(lines.bytes, [&](auto b) {
            using L = Lanes<decltype(t), b()>;
            const int vec = together(op->y, op->ldy, op->y_type, L::kOf);
            auto go = [&](auto kernel) { kernel<<<ctas_for(lines.warps), kTableThreads, 0, static_cast<cudaStream_t>(stream)>>>(*op, vec); };
            constexpr int kFew = b() == 32 || b() == 0 ? kEmbedAhead : kFewAhead;
            if (op->slots <= kEmbedAhead && !lines.few)
                embed_short_kernel<decltype(t), b()><<<ctas_for((op->rows + lists - 1ll) / lists * lines.across), kTableThreads, 0, static_cast<cudaStream_t>(stream)>>>(*op, lists, vec);
            else if (lines.few)
                go(embed_kernel<decltype(t), b(), kFew>);
            else
                go(embed_kernel<decltype(t), b(), kEmbedAhead>);
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
    if (op->rows == 0) return zeros(op, s);
    if (few_rows(op)) {
        const Few few = few_of(op);
        if ((int64_t)few.chunks * few.across > INT32_MAX) return fail(B200_ERR_UNSUPPORTED, "%s: %d lists, %d columns are too many", who, op->rows, op->cols);
        int rc = 0;
        with_float(op->dy_type, [&](auto t) {
            with_bytes(few.bytes, [&](auto b) {
                if constexpr (b() != 32) rc = few_rows_gradient<decltype(t), b()>(op, few, s);
            });
        });
        return rc;
    }
    char* base = static_cast<char*>(op->workspace);
    const Sorting sort = sorting_of(op);
    if (sort.places)
        if (int rc = zeros(op, s)) return rc;
    int2* pairs[2] = {reinterpret_cast<int2*>(base + space.pairs), reinterpret_cast<int2*>(base + space.more_pairs)};
    int* start = sort.places ? nullptr : reinterpret_cast<int*>(base + space.start);
    int* numbers = reinterpret_cast<int*>(base + space.numbers);
    const Long l{numbers, reinterpret_cast<Piece8*>(base + space.pieces), reinterpret_cast<int*>(base + space.done), space.piece, space.lines.across};
    SortPass p{};
    p.ids = op->ids, p.ldids = op->ldids, p.slots = (uint32_t)op->slots, p.wide = op->wide_ids, p.n = op->n;
    p.count = (uint32_t)sort.count, p.tiles = sort.tiles, p.bits = sort.bits, p.to = pairs[0];
    if (sort.one()) {
        const size_t shared = kSortOne * 8 + (((size_t)32 << sort.bits) + 32) * 4;
        static std::atomic<uint64_t> allowed;  // a bit per device
        if (device >= 64 || !(allowed >> device & 1)) {
            OP_CK(cudaFuncSetAttribute(sort_one_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortOne * 8 + 32 * 257 * 4));
            if (device < 64) allowed |= (uint64_t)1 << device;
        }
        sort_one_kernel<<<1, kOneThreads, shared, s>>>(p, sort.passes, start, numbers + 1, l);
        OP_CK(cudaGetLastError());
    } else {
        p.counts = reinterpret_cast<int*>(base + space.counts);
        p.there = numbers + 1;
        for (int k = 0; k < sort.passes; k++) {
            p.to = pairs[k & 1];
            p.shift = k * sort.bits;
            OP_CK(launch_step(k > 0, pass_count_kernel, sort.tiles, kSortThreads, 0, s, p, numbers));
            OP_CK(launch_step(true, pass_sum_kernel, ((1 << sort.bits) + kSortWarps - 1) / kSortWarps, kSortThreads, 0, s, p.counts, 1 << sort.bits, sort.tiles));
            OP_CK(launch_step(true, pass_place_kernel, sort.tiles, kSortThreads, 0, s, p));
            p.from = p.to;
        }
        if (sort.places) {
            OP_CK(launch_step(true, list_long_places_kernel, (unsigned)((sort.count + kTableThreads - 1) / kTableThreads), kTableThreads, 0, s, p.to, p.there, l));
        } else {
            OP_CK(launch_step(true, starts_kernel, (unsigned)((sort.count + kTableThreads * kStartsEach) / (kTableThreads * kStartsEach)), kTableThreads, 0, s, p.to, p.there, op->n, start));
            OP_CK(launch_step(true, list_long_kernel, (unsigned)((op->n + kTableThreads - 1ll) / kTableThreads), kTableThreads, 0, s, start, op->n, l));
        }
    }
    TableGrad g{*op, p.to, start, numbers + 1, l, reinterpret_cast<float*>(base + space.parts), space.ldp, space.cuts, 0};
    cudaError_t rc = cudaSuccess;
    with_float(op->dy_type, [&](auto t) {
        with_bytes(space.lines.bytes, [&](auto b) {
            using L = Lanes<decltype(t), b()>;
            g.vec = together(op->dtable, op->lddt, op->dtable_type, L::kOf);
            auto go = [&](auto kernel) { rc = launch_step(true, kernel, ctas_for(space.lines.warps), kTableThreads, 0, s, g); };
            constexpr int kFew = b() == 32 || b() == 0 ? kGradAhead : kFewAhead;
            if (space.lines.few)
                sort.places ? go(embed_backward_kernel<decltype(t), b(), kFew, true>) : go(embed_backward_kernel<decltype(t), b(), kFew, false>);
            else
                sort.places ? go(embed_backward_kernel<decltype(t), b(), kGradAhead, true>) : go(embed_backward_kernel<decltype(t), b(), kGradAhead, false>);
        });
    });
    OP_CK(rc);
    return 0;
}

}  // extern "C"
