// Operator-level entry point of the norm of many tensors and its limit: b200_op_clip_gradients.
#include <algorithm>
#include <vector>

#include "kernels_clip.cuh"
#include "op_call.h"

namespace {

using namespace b200;

int64_t chunks_of(const b200_gradient& t) { return (t.n + kClipChunk - 1) / kClipChunk; }
constexpr int64_t kChunksMost = INT32_MAX - 65536;  // of a launch

int check_clip(const b200_clip_op* op, const char* who) {
    if (!op) return fail(B200_ERR_ARG, "%s: null operator description", who);
    if (op->count < 0) return fail(B200_ERR_ARG, "%s: %d tensors", who, op->count);
    if (op->count && !op->gradients) return fail(B200_ERR_ARG, "%s: gradients is NULL", who);
    for (int k = 0; k < op->count; k++) {
        const b200_gradient& t = op->gradients[k];
        if (!is_float(t.type)) return fail(B200_ERR_UNSUPPORTED, "%s: type %d of gradient %d", who, t.type, k);
        if (t.n < 0 || t.n > kChunksMost * kClipChunk) return fail(B200_ERR_ARG, "%s: %lld elements of gradient %d", who, (long long)t.n, k);
    }
    return 0;
}
// The tensors, kClipMost at a time: f(the first of a launch, the one behind its last)
template <class F>
int64_t batches(const b200_clip_op* op, F f) {
    int64_t launches = 0;
    for (int first = 0, k = 0; first < op->count; first = k, launches++) {
        int64_t chunks = 0;
        for (; k < op->count && k < first + kClipMost && chunks + chunks_of(op->gradients[k]) <= kChunksMost; k++) chunks += chunks_of(op->gradients[k]);
        f(first, k);
    }
    return launches;
}
int64_t clip_bytes(const b200_clip_op* op) { return std::max<int64_t>(1, batches(op, [](int, int) {})) * kClipCtas * 8; }
ClipBatch batch_of(const b200_clip_op* op, int first, int last) {
    ClipBatch b;
    b.count = b.chunks = 0;
    for (int k = first; k < last; k++) {
        const b200_gradient& t = op->gradients[k];
        if (!t.n) continue;
        const int at = b.count++;
        b.g[at] = t.g, b.out[at] = t.out, b.n[at] = t.n, b.first[at] = b.chunks, b.type[at] = (uint8_t)t.type;
        b.vec[at] = ((uintptr_t)t.g | (uintptr_t)t.out) % 16 == 0;
        b.chunks += (int)chunks_of(t);
    }
    return b;
}

double limit_of(const b200_clip_op* op) { return (double)op->max_norm + op->max_norm_low; }

// Whether what is written overlaps what is read or written elsewhere; a tensor may be scaled in place.
int check_overlaps(const b200_clip_op* op, const char* who) {
    struct Range {
        uintptr_t from, to;
        int tensor;
    };
    std::vector<Range> outs;
    outs.reserve(op->count);
    for (int k = 0; k < op->count; k++) {
        const b200_gradient& t = op->gradients[k];
        if (t.out && t.n) outs.push_back({(uintptr_t)t.out, (uintptr_t)t.out + t.n * type_bytes(t.type), k});
    }
    std::sort(outs.begin(), outs.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    for (size_t k = 1; k < outs.size(); k++)
        if (outs[k].from < outs[k - 1].to) return fail(B200_ERR_ARG, "%s: outputs %d and %d overlap", who, outs[k - 1].tensor, outs[k].tensor);
    if (outs.empty()) return 0;
    for (int k = 0; k < op->count; k++) {
        const b200_gradient& t = op->gradients[k];
        if (!t.n) continue;
        const uintptr_t from = (uintptr_t)t.g, to = from + t.n * type_bytes(t.type);
        // (outputs do not overlap: those that this one meets are neighbours, from the last that begins before its end on backwards)
        auto at = std::lower_bound(outs.begin(), outs.end(), to, [](const Range& a, uintptr_t end) { return a.from < end; });
        while (at != outs.begin() && (--at)->to > from)
            if (at->tensor != k || at->from != from) return fail(B200_ERR_ARG, "%s: output %d overlaps gradient %d", who, at->tensor, k);
    }
    return 0;
}

}  // namespace

extern "C" {

int b200_op_clip_gradients_workspace(const b200_clip_op* op, int64_t* bytes) {
    if (int rc = check_clip(op, "op_clip_gradients")) return rc;
    if (!bytes) return fail(B200_ERR_ARG, "op_clip_gradients: null result");
    *bytes = clip_bytes(op);
    return 0;
}

int b200_op_clip_gradients(int device, void* stream, const b200_clip_op* op) try {
    const char* who = "op_clip_gradients";
    if (int rc = check_clip(op, who)) return rc;
    bool writes = false;
    for (int k = 0; k < op->count; k++) {
        const b200_gradient& t = op->gradients[k];
        if (t.n && !t.g) return fail(B200_ERR_ARG, "%s: gradient %d is NULL", who, k);
        if (((uintptr_t)t.g | (uintptr_t)t.out) % type_bytes(t.type)) return fail(B200_ERR_ARG, "%s: gradient %d is not aligned to its elements", who, k);
        writes |= t.n && t.out;
    }
    if (writes && !(limit_of(op) >= 0)) return fail(B200_ERR_ARG, "%s: max_norm must not be negative", who);
    if (int rc = check_overlaps(op, who)) return rc;
    if (int rc = check_floats(who, "norm", op->norm)) return rc;
    if (int rc = check_workspace(who, op->workspace, op->workspace_bytes, clip_bytes(op))) return rc;
    OnDevice on(device);
    OP_CK(on.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* sums = static_cast<double*>(op->workspace);
    ClipTotal total{sums, 0, limit_of(op), op->norm};
    cudaError_t rc = cudaSuccess;
    batches(op, [&](int first, int last) {
        const ClipBatch b = batch_of(op, first, last);
        if (!b.chunks || rc != cudaSuccess) return;
        const int ctas = std::min(b.chunks, kClipCtas);
        squares_kernel<<<ctas, kClipThreads, 0, s>>>(b, sums + total.n_sums);
        rc = cudaGetLastError();
        total.n_sums += ctas;
    });
    OP_CK(rc);
    if (!writes) {
        OP_CK(launch_step(total.n_sums > 0, norm_kernel, 1, kClipThreads, 0, s, total));
        return 0;
    }
    bool follows = true;  // (the kernel before it is the sums')
    batches(op, [&](int first, int last) {
        const ClipBatch b = batch_of(op, first, last);
        if (!b.chunks || rc != cudaSuccess) return;
        rc = launch_step(follows, clip_kernel, std::min(b.chunks, kClipCtas), kClipThreads, 0, s, b, total);
        total.norm = nullptr;
        follows = false;
    });
    OP_CK(rc);
    return 0;
} catch (const std::exception& e) {
    return b200::fail(B200_ERR_STATE, "op_clip_gradients: %s", e.what());
}

}  // extern "C"
