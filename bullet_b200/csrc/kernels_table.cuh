// Rows of a table that lists of ids name: their sums per list, and the gradient, the sums of the lists' gradients per row of the table.
//
// The gradient's sums are taken in the order of the lists, so ids are sorted first, stably: by counting, a digit of up to eight bits a pass
// (pass_count_kernel, pass_scan_kernel, pass_place_kernel).  Then a thread takes eight columns of one table row and adds the rows up that its
// stretch of the sorted ids names.  Stretches of more than kStretch are cut at multiples of kStretch of the sorted order, whose sums go to
// memory and are joined in order: a piece has parts of two such stretches at most, its first id's and its last one's.
#pragma once
#include <cuda_runtime.h>

#include "kernels_four.cuh"
#include "launch.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kTableThreads = 256;

// ---- sums of rows

// An id, or -1 for one that names no row.
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i, int wide, int64_t n) {
    const int64_t id = wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
    return id >= 0 && id < n ? id : -1;
}

template <bool VEC, class T>
struct Row8 {
    T v[8];
    __device__ __forceinline__ void load(const T* row, int64_t first, int64_t cols) {
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) reinterpret_cast<uint4*>(v)[k] = __ldg(reinterpret_cast<const uint4*>(row + first) + k);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = first + k < cols ? __ldg(row + first + k) : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void add(float (&sum)[8]) const {
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] += to_float(v[k]);
    }
};
template <bool VEC>
__device__ __forceinline__ void store_typed(void* y, int64_t row_at, int64_t first, int64_t cols, int type, const float (&v)[8]) {
    if (type == B200_TYPE_F32)
        store_values<VEC>(static_cast<float*>(y) + row_at, first, cols, v);
    else if (type == B200_TYPE_BF16)
        store_values<VEC>(static_cast<bf16*>(y) + row_at, first, cols, v);
    else
        store_values<VEC>(static_cast<f16*>(y) + row_at, first, cols, v);
}

constexpr int kSlotsAhead = 8;
// A thread takes eight columns of a list.
template <class T, bool VEC>
static __global__ void __launch_bounds__(kTableThreads) embed_kernel(b200_embed_op a) {
    Place p((int64_t)blockIdx.x * kTableThreads + threadIdx.x, (int64_t)gridDim.x * kTableThreads, (a.cols + 7) / 8);
    const T* table = static_cast<const T*>(a.table);
    for (; p.row < a.rows; p.next()) {
        float sum[8] = {};
        for (int s = 0; s < a.slots; s += kSlotsAhead) {
            int64_t id[kSlotsAhead];
            Row8<VEC, T> row[kSlotsAhead];
#pragma unroll
            for (int k = 0; k < kSlotsAhead; k++) id[k] = s + k < a.slots ? id_at(a.ids, p.row * a.ldids + s + k, a.wide_ids, a.n) : -1;
#pragma unroll
            for (int k = 0; k < kSlotsAhead; k++)
                if (id[k] >= 0) row[k].load(table + id[k] * a.ldt, p.at * 8, a.cols);
#pragma unroll
            for (int k = 0; k < kSlotsAhead; k++)
                if (id[k] >= 0) row[k].add(sum);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] *= a.scale;
        store_typed<VEC>(a.y, p.row * a.ldy, p.at * 8, a.cols, a.y_type, sum);
    }
}

// ---- ids sorted

constexpr int kSortThreads = 256, kSortEach = 16, kSortTile = kSortThreads * kSortEach, kSortWarps = kSortThreads / 32;
struct SortPass {
    const void* ids;       // the first pass's, in lists
    int64_t ldids;
    int slots, wide, n;
    const int2* from;      // the later ones': (id, list)
    int2* to;
    int64_t count;         // of ids
    int shift, bits;       // of the digit
    int* counts;           // [1 << bits][tiles]
    int tiles;
};
// Element i of a pass: an id (n: none) and the list that it stands in.
__device__ __forceinline__ int2 sort_element(const SortPass& p, int64_t i) {
    if (p.from) return __ldcg(p.from + i);
    const int64_t list = i / p.slots, id = id_at(p.ids, list * p.ldids + i % p.slots, p.wide, p.n);
    return make_int2(id < 0 ? p.n : (int)id, (int)list);
}
__device__ __forceinline__ int sort_digit(const SortPass& p, int id) { return id >> p.shift & ((1 << p.bits) - 1); }

static __global__ void __launch_bounds__(kSortThreads) pass_count_kernel(SortPass p) {
    __shared__ int count[256];
    step_begin(nullptr);
    count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kSortTile;
#pragma unroll 4
    for (int k = 0; k < kSortEach; k++) {
        const int64_t i = first + k * kSortThreads + threadIdx.x;
        if (i < p.count) atomicAdd(count + sort_digit(p, sort_element(p, i).x), 1);
    }
    __syncthreads();
    if (threadIdx.x < 1 << p.bits) p.counts[(int64_t)threadIdx.x * p.tiles + blockIdx.x] = count[threadIdx.x];
}
// Counts to where each tile's first element of each digit goes: one CTA.
static __global__ void __launch_bounds__(1024) pass_scan_kernel(int* counts, int64_t n) {
    __shared__ int sums[32];
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int before = 0;
    for (int64_t base = 0; base < n; base += 4096) {
        const int64_t i = base + threadIdx.x * 4;
        int v[4], own = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = i + k < n ? __ldcg(counts + i + k) : 0;
            own += v[k];
        }
        int run = own;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int u = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += u;
        }
        if (lane == 31) sums[warp] = run;
        __syncthreads();
        if (warp == 0) {
            int w = sums[lane];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += u;
            }
            sums[lane] = w;
        }
        __syncthreads();
        int at = before + (warp ? sums[warp - 1] : 0) + run - own;
        before += sums[31];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (i + k < n) counts[i + k] = at;
            at += v[k];
        }
        __syncthreads();
    }
}
// A warp takes kSortEach x 32 neighbours in order: an element's rank among its warp's of the same digit, then the warps before, then the tiles.
static __global__ void __launch_bounds__(kSortThreads) pass_place_kernel(SortPass p) {
    __shared__ int count[kSortWarps][256];
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = threadIdx.x; k < kSortWarps * 256; k += kSortThreads) count[k >> 8][k & 255] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kSortTile + warp * 32 * kSortEach + lane;
    int2 element[kSortEach];
    int rank[kSortEach];
#pragma unroll
    for (int k = 0; k < kSortEach; k++) element[k] = first + k * 32 < p.count ? sort_element(p, first + k * 32) : make_int2(-1, 0);
#pragma unroll
    for (int k = 0; k < kSortEach; k++) {
        const bool here = first + k * 32 < p.count;
        const int digit = here ? sort_digit(p, element[k].x) : 256 + lane;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (here) rank[k] = count[warp][digit] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (here && (same >> lane) == 1u) count[warp][digit] = rank[k] + 1;  // (the last of them)
        __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < 1 << p.bits) {
        int at = __ldcg(p.counts + (int64_t)threadIdx.x * p.tiles + blockIdx.x);
        for (int w = 0; w < kSortWarps; w++) {
            const int own = count[w][threadIdx.x];
            count[w][threadIdx.x] = at;
            at += own;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; k++)
        if (first + k * 32 < p.count) p.to[count[warp][sort_digit(p, element[k].x)] + rank[k]] = element[k];
}

// start[t]: where row t's stretch of the sorted ids begins, t up to n.  A thread per place between two ids fills in the rows that begin there; where
// there are many (ids far apart) its warp does.
static __global__ void __launch_bounds__(kTableThreads) stretches_kernel(const int2* sorted, int64_t count, int n, int* start) {
    step_begin(nullptr);
    const int64_t i = (int64_t)blockIdx.x * kTableThreads + threadIdx.x;
    const int lane = threadIdx.x & 31;
    const int before = i == 0 || i > count ? -1 : __ldcg(sorted + i - 1).x, id = i < count ? __ldcg(sorted + i).x : n;
    const int gap = i <= count ? id - before : 0;
    if (gap > 0 && gap <= 32)
        for (int t = before + 1; t <= id; t++) start[t] = (int)i;
    for (unsigned wide = __ballot_sync(0xffffffffu, gap > 32); wide; wide &= wide - 1) {
        const int from = __ffs(wide) - 1;
        const int b = __shfl_sync(0xffffffffu, before, from), e = __shfl_sync(0xffffffffu, id, from);
        const int at = (int)(i - lane + from);
        for (int64_t t = b + 1ll + lane; t <= e; t += 32) start[t] = at;
    }
}

// ---- the gradient

constexpr int kStretch = 64, kRowsAhead = 8;
struct TableGrad {
    b200_embed_grad_op a;
    const int2* sorted;
    const int* start;
    float* parts;  // [2][pieces][ldp]: of a piece's first id, and of its last one where that is another
    int64_t ldp, pieces;
};
// The sum of what stretch [from, to) of the sorted ids names.
template <class T, bool VEC>
__device__ __forceinline__ void add_stretch(const TableGrad& g, int from, int to, int64_t first, float (&sum)[8]) {
    const T* dy = static_cast<const T*>(g.a.dy);
    for (int s = from; s < to; s += kRowsAhead) {
        Row8<VEC, T> row[kRowsAhead];
        int list[kRowsAhead];
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++) list[k] = s + k < to ? __ldcg(&g.sorted[s + k].y) : -1;
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++)
            if (list[k] >= 0) row[k].load(dy + list[k] * g.a.lddy, first, g.a.cols);
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++)
            if (list[k] >= 0) row[k].add(sum);
    }
}
// Rows of the table, then pieces.
template <class T, bool VEC>
static __global__ void __launch_bounds__(kTableThreads) embed_backward_kernel(TableGrad g) {
    step_begin(nullptr);
    Place p((int64_t)blockIdx.x * kTableThreads + threadIdx.x, (int64_t)gridDim.x * kTableThreads, (g.a.cols + 7) / 8);
    for (; p.row < g.a.n + g.pieces; p.next()) {
        const int64_t first = p.at * 8;
        if (p.row < g.a.n) {
            const int from = __ldcg(g.start + p.row), to = __ldcg(g.start + p.row + 1);
            if (to - from > kStretch) continue;
            float sum[8] = {};
            add_stretch<T, VEC>(g, from, to, first, sum);
#pragma unroll
            for (int k = 0; k < 8; k++) sum[k] *= g.a.scale;
            store_typed<VEC>(g.a.dtable, p.row * g.a.lddt, first, g.a.cols, g.a.dtable_type, sum);
        } else {
            const int64_t piece = p.row - g.a.n;
            const int all = __ldcg(g.start + g.a.n), begin = (int)(piece * kStretch), end = min(begin + kStretch, all);
            if (begin >= end) continue;
            const int id[2] = {__ldcg(&g.sorted[begin].x), __ldcg(&g.sorted[end - 1].x)};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (h && id[1] == id[0]) break;
                const int from = __ldcg(g.start + id[h]), to = __ldcg(g.start + id[h] + 1);
                if (to - from <= kStretch) continue;
                float sum[8] = {};
                add_stretch<T, VEC>(g, max(from, begin), min(to, end), first, sum);
                store_values<true>(g.parts + (h * g.pieces + piece) * g.ldp, first, g.a.cols, sum);
            }
        }
    }
}
// Rows with stretches that were cut.
template <bool VEC>
static __global__ void __launch_bounds__(kTableThreads) embed_join_kernel(TableGrad g) {
    step_begin(nullptr);
    Place p((int64_t)blockIdx.x * kTableThreads + threadIdx.x, (int64_t)gridDim.x * kTableThreads, (g.a.cols + 7) / 8);
    for (; p.row < g.a.n; p.next()) {
        const int from = __ldcg(g.start + p.row), to = __ldcg(g.start + p.row + 1);
        if (to - from <= kStretch) continue;
        const int64_t first = p.at * 8;
        const int piece0 = from / kStretch, piece1 = (to - 1) / kStretch;
        float sum[8] = {};
#pragma unroll 4
        for (int piece = piece0; piece <= piece1; piece++) {
            const bool last = piece == piece0 && __ldcg(&g.sorted[piece * kStretch].x) != p.row;  // (it begins behind the piece's first id)
            const float* part = g.parts + ((last ? g.pieces : 0) + piece) * g.ldp + first;
            const float4 u = __ldcg(reinterpret_cast<const float4*>(part)), v = __ldcg(reinterpret_cast<const float4*>(part) + 1);
            sum[0] += u.x, sum[1] += u.y, sum[2] += u.z, sum[3] += u.w, sum[4] += v.x, sum[5] += v.y, sum[6] += v.z, sum[7] += v.w;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] *= g.a.scale;
        store_typed<VEC>(g.a.dtable, p.row * g.a.lddt, first, g.a.cols, g.a.dtable_type, sum);
    }
}

}  // namespace b200
