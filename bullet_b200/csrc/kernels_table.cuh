// Rows of a table that lists of ids name: their sums per list, and the gradient, the sums of the lists' gradients per row of the table.
//
// Bound by L2's way to the SMs (16384 lists of 17 rows of 2 KB are 590 MB out of a table of 25, in 39 us), with few lists by latency.  A warp takes a list, or a row of
// the table, and the columns that its lanes cover with 32 bytes each, for what a row's index and address cost: with 16, 57 us.  (Fewer in narrow matrices; single elements
// 32 apart where rows do not start on 16 bytes.)
// Its lanes load 32 indices side by side and hand them round, and four to sixteen rows are on their way at a time.
//
// The gradient's sums are taken in the order of the lists, so ids are sorted first, stably, by counting digits of up to eight bits: one CTA for up to kSortOne
// ids, else three kernels a pass.  Ids that name no row are left out by the first pass.  Then a warp adds up the rows that a table row's stretch of the
// sorted ids names.  Stretches of more than kLongest are listed and cut into pieces, whose sums go to memory and are joined in order.
// A table of more rows than there are ids is set to 0 first, and a warp looks at each of the sorted ids for whether a stretch begins there, so that rows without ids cost no
// more than their zeros.
#pragma once
#include <cuda_runtime.h>

#include "kernels_four.cuh"
#include "launch.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kTableThreads = 256;
// Rows on their way in a warp.  Warps that hide each other's latency count for more than rows in one: 16384 x 32 features of 1024 columns, two rows of 32 bytes a lane and
// 32 warps of an SM 43 us, four 39; their gradient, four rows and 24 warps (80 bytes of a thread's registers spilt) 82, 32 (and more spilt) 96, two rows and 32 83, six and
// 24 92; by 16 bytes four rows and 32 warps 96, eight 102, four and 40 103.
// So many warps as fill the GPU twice over or fewer take sixteen rows of 16 bytes each.
constexpr int kEmbedAhead = 4, kGradAhead = 4, kFewAhead = 16;

// A warp's place: one of up to 2^32 rows, and of `across` chunks of its columns; next() as many on as there are warps.
struct WarpPlace {
    uint32_t row, rows_on;
    int at, on, across;
    __device__ explicit WarpPlace(int across_) : across(across_) {
        const uint32_t warps = gridDim.x * (kTableThreads / 32), own = blockIdx.x * (kTableThreads / 32) + (threadIdx.x >> 5);  // (a grid has few)
        row = own / across, at = (int)(own % across), rows_on = warps / across, on = (int)(warps % across);
    }
    __device__ __forceinline__ void next() {
        row += rows_on, at += on;
        if (at >= across) at -= across, row++;
    }
};

// ---- sums of rows

// An id, or -1 for one that names no row.
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i, int wide, int64_t n) {
    const int64_t id = wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
    return id >= 0 && id < n ? id : -1;
}

// sum += v, a value of 16 bits, by one instruction (the same sum as of the value in 32 bits)
template <class T>
__device__ __forceinline__ void add_half(float& sum, uint16_t v) {
    if constexpr (std::is_same_v<T, bf16>)
        asm("add.rn.f32.bf16 %0, %1, %0;" : "+f"(sum) : "h"(v));
    else
        asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(sum) : "h"(v));
}
// A lane's columns of a warp's: BYTES side by side, with 32 twice 16 half a warp's columns apart, or with 0 as many single elements as 16 bytes hold, 32 apart.
template <class T, int BYTES>
struct Lanes {
    static constexpr int kParts = BYTES == 32 ? 2 : 1, kBytes = BYTES == 32 || BYTES == 0 ? 16 : BYTES;  // of a part
    static constexpr int kOf = kBytes / (int)sizeof(T), kEach = kParts * kOf, kWarp = 32 * kEach;
    static __device__ __forceinline__ int64_t first(int64_t chunk) { return chunk * kWarp + (threadIdx.x & 31) * (BYTES ? kOf : 1); }
    static __device__ __forceinline__ int64_t column(int64_t at, int k) { return at + (BYTES ? k / kOf * 32 * kOf + k % kOf : 32 * k); }
    T v[kEach];
    __device__ __forceinline__ void load(const T* row, int64_t at, int64_t cols) {
#pragma unroll
        for (int part = 0; part < kParts; part++) {
            const T* from = row + column(at, part * kOf);
            T* to = v + part * kOf;
            if constexpr (BYTES == 0) {
#pragma unroll
                for (int k = 0; k < kEach; k++)
                    if (column(at, k) < cols) v[k] = __ldg(row + column(at, k));
            } else if (column(at, part * kOf) < cols) {
                if constexpr (kBytes == 16)
                    *reinterpret_cast<uint4*>(to) = __ldg(reinterpret_cast<const uint4*>(from));
                else if constexpr (kBytes == 8)
                    *reinterpret_cast<uint2*>(to) = __ldg(reinterpret_cast<const uint2*>(from));
                else
                    *reinterpret_cast<uint32_t*>(to) = __ldg(reinterpret_cast<const uint32_t*>(from));
            }
        }
    }
    __device__ __forceinline__ void add(float (&sum)[kEach]) const {
        if constexpr (sizeof(T) == 2 && kEach > 1) {
#pragma unroll
            for (int k = 0; k < kEach; k += 2) {
                uint16_t low, high;
                memcpy(&low, v + k, 2);
                memcpy(&high, v + k + 1, 2);
                add_half<T>(sum[k], low);
                add_half<T>(sum[k + 1], high);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kEach; k++) sum[k] += to_float(v[k]);
        }
    }
};
// kEach sums to a row of `type`, whose elements start where those of T did (VEC: on a part's elements together).
template <class T, int BYTES, bool VEC>
__device__ __forceinline__ void store_sums(void* y, int64_t row_at, int64_t at, int64_t cols, int type, const float (&v)[Lanes<T, BYTES>::kEach]) {
    using L = Lanes<T, BYTES>;
    constexpr int kOf = L::kOf;
#pragma unroll
    for (int part = 0; part < L::kParts; part++) {
        const int64_t column = L::column(at, part * kOf);
        const int first = part * kOf;
        if constexpr (BYTES != 0 && VEC && kOf > 1) {
            if (column >= cols) continue;
            if (type == B200_TYPE_F32) {
                float* to = static_cast<float*>(y) + row_at + column;
                if constexpr (kOf >= 4) {
#pragma unroll
                    for (int k = 0; k < kOf; k += 4) *reinterpret_cast<float4*>(to + k) = make_float4(v[first + k], v[first + k + 1], v[first + k + 2], v[first + k + 3]);
                } else {
                    *reinterpret_cast<float2*>(to) = make_float2(v[first], v[first + 1]);
                }
            } else {
                uint32_t w[kOf / 2];
#pragma unroll
                for (int k = 0; k < kOf / 2; k++) w[k] = type == B200_TYPE_BF16 ? pack2<bf16>(v[first + 2 * k], v[first + 2 * k + 1]) : pack2<f16>(v[first + 2 * k], v[first + 2 * k + 1]);
                uint16_t* to = static_cast<uint16_t*>(y) + row_at + column;
                if constexpr (kOf == 8)
                    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                else if constexpr (kOf == 4)
                    *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
                else
                    *reinterpret_cast<uint32_t*>(to) = w[0];
            }
        } else {
#pragma unroll
            for (int k = first; k < first + kOf; k++)
                if (L::column(at, k) < cols) store_value(y, row_at + L::column(at, k), type, v[k]);
        }
    }
}
// Adds the rows that the lanes in `mask` name, in the lanes' order.
template <class T, int BYTES, int AHEAD>
__device__ __forceinline__ void add_named(const T* rows, int64_t ld, int64_t at, int64_t cols, int index, unsigned mask, float (&sum)[Lanes<T, BYTES>::kEach]) {
    while (mask) {
        Lanes<T, BYTES> row[AHEAD];
        const int there = min(AHEAD, __popc(mask));
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int64_t r = __shfl_sync(0xffffffffu, index, __ffs(mask) - 1);  // (0 left: lane 31's, and not used)
            mask &= mask - 1;
            if (k < there) row[k].load(rows + r * ld, at, cols);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (k < there) row[k].add(sum);
    }
}
// ... that the first `lanes` of them name: a sum's instructions count as well (the features' gradient, with four rows on their way, 110 us by masks, 96 so).
template <class T, int BYTES, int AHEAD>
__device__ __forceinline__ void add_first(const T* rows, int64_t ld, int64_t at, int64_t cols, int index, int lanes, float (&sum)[Lanes<T, BYTES>::kEach]) {
    for (int j = 0; j < lanes; j += AHEAD) {
        Lanes<T, BYTES> row[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int64_t r = __shfl_sync(0xffffffffu, index, j + k);  // (past the last: some lane's, and not used)
            if (j + k < lanes) row[k].load(rows + r * ld, at, cols);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (j + k < lanes) row[k].add(sum);
    }
}

// VEC: a row of y takes a lane's elements together.
template <class T, int BYTES, int AHEAD>
static __global__ void __launch_bounds__(kTableThreads, AHEAD == kFewAhead || BYTES == 0 ? 2 : 4) embed_kernel(b200_embed_op a, int vec) {
    using L = Lanes<T, BYTES>;
    const int lane = threadIdx.x & 31;
    WarpPlace p((int)((a.cols + L::kWarp - 1ll) / L::kWarp));
    for (; p.row < (uint32_t)a.rows; p.next()) {
        const int64_t at = L::first(p.at);
        float sum[L::kEach] = {};
        for (int s = 0; s < a.slots; s += 32) {
            const int64_t id = s + lane < a.slots ? id_at(a.ids, p.row * a.ldids + s + lane, a.wide_ids, a.n) : -1;
            add_named<T, BYTES, AHEAD>(static_cast<const T*>(a.table), a.ldt, at, a.cols, (int)id, __ballot_sync(0xffffffffu, id >= 0), sum);
        }
#pragma unroll
        for (int k = 0; k < L::kEach; k++) sum[k] *= a.scale;
        if (vec)
            store_sums<T, BYTES, true>(a.y, p.row * a.ldy, at, a.cols, a.y_type, sum);
        else
            store_sums<T, BYTES, false>(a.y, p.row * a.ldy, at, a.cols, a.y_type, sum);
    }
}
// Lists of up to kEmbedAhead ids: a warp takes `lists` of them, as many as its lanes have room for or fewer, and of these as many at a time as have kEmbedAhead ids together.  (One
// id each, 131072 x 1024 bf16: of 12288 rows 63 us, a list at a time 147; of 8 rows 51, with 41 of them what HBM takes to write y.)
template <class T, int BYTES>
static __global__ void __launch_bounds__(kTableThreads, BYTES == 0 ? 2 : 4) embed_short_kernel(b200_embed_op a, int lists, int vec) {
    using L = Lanes<T, BYTES>;
    const int lane = threadIdx.x & 31, at_once = kEmbedAhead / a.slots;
    WarpPlace p((int)((a.cols + L::kWarp - 1ll) / L::kWarp));
    for (; (int64_t)p.row * lists < a.rows; p.next()) {
        const int64_t at = L::first(p.at), first = (int64_t)p.row * lists;
        const int there = (int)min((int64_t)lists, a.rows - first);
        const int list = lane / a.slots;
        const int id = list < there ? (int)id_at(a.ids, (first + list) * a.ldids + lane % a.slots, a.wide_ids, a.n) : -1;
        for (int l0 = 0; l0 < there; l0 += at_once) {
            L row[kEmbedAhead];
            int named = 0;  // a bit each
#pragma unroll
            for (int k = 0; k < kEmbedAhead; k++) {
                const int r = __shfl_sync(0xffffffffu, id, (l0 * a.slots + k) & 31);
                if (k < at_once * a.slots && r >= 0 && l0 * a.slots + k < 32) {
                    row[k].load(static_cast<const T*>(a.table) + r * a.ldt, at, a.cols);
                    named |= 1 << k;
                }
            }
            float sum[L::kEach] = {};
            int slot = 0, l = l0;
#pragma unroll
            for (int k = 0; k < kEmbedAhead; k++) {
                if (named >> k & 1) row[k].add(sum);
                if (++slot == a.slots) {
                    if (l < there && l < l0 + at_once) {
#pragma unroll
                        for (int i = 0; i < L::kEach; i++) sum[i] *= a.scale;
                        if (vec)
                            store_sums<T, BYTES, true>(a.y, (first + l) * a.ldy, at, a.cols, a.y_type, sum);
                        else
                            store_sums<T, BYTES, false>(a.y, (first + l) * a.ldy, at, a.cols, a.y_type, sum);
                    }
#pragma unroll
                    for (int i = 0; i < L::kEach; i++) sum[i] = 0.f;
                    slot = 0, l++;
                }
            }
        }
    }
}


// ---- ids sorted

constexpr int kSortThreads = 256, kSortEach = 8, kSortTile = kSortThreads * kSortEach, kSortWarps = kSortThreads / 32;
struct SortPass {
    const void* ids;       // the first pass's, in lists
    int64_t ldids;
    uint32_t slots;
    int wide, n;
    const int2* from;      // the later ones': (id, list)
    int2* to;
    uint32_t count;        // of ids, there or not
    int* there;            // how many are: left by the first pass, which the later ones read
    int shift, bits;       // of the digit
    int* counts;           // [1 << bits][tiles], and behind them [1 << bits]: of a digit all
    int tiles;
};
// Elements first, first + apart, ... of a pass's `all`, (id, list), loaded together; (-1, ..) for an id that names no row and past the last one.
template <int EACH>
__device__ __forceinline__ void sort_elements(const SortPass& p, uint32_t first, uint32_t apart, uint32_t all, int2 (&element)[EACH]) {
#pragma unroll
    for (int k = 0; k < EACH; k++) element[k] = make_int2(-1, 0);
    if (first >= all) return;
    if (p.from) {
#pragma unroll
        for (int k = 0; k < EACH; k++) element[k] = __ldcg(p.from + min(first + k * apart, all - 1));
    } else {
        int64_t at[EACH], id[EACH];
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const uint32_t i = min(first + k * apart, all - 1), list = p.slots == 1 ? i : i / p.slots;
            element[k].y = (int)list, at[k] = list * p.ldids + (i - list * p.slots);
        }
        if (p.wide) {
#pragma unroll
            for (int k = 0; k < EACH; k++) id[k] = static_cast<const int64_t*>(p.ids)[at[k]];
        } else {
#pragma unroll
            for (int k = 0; k < EACH; k++) id[k] = static_cast<const int32_t*>(p.ids)[at[k]];
        }
#pragma unroll
        for (int k = 0; k < EACH; k++) element[k].x = id[k] >= 0 && id[k] < p.n ? (int)id[k] : -1;
    }
#pragma unroll
    for (int k = 0; k < EACH; k++)
        if (first + k * apart >= all) element[k].x = -1;
}
__device__ __forceinline__ int sort_digit(const SortPass& p, int id) { return id >> p.shift & ((1 << p.bits) - 1); }

static __global__ void __launch_bounds__(kSortThreads) pass_count_kernel(SortPass p, int* cleared) {
    __shared__ int count[256];
    step_begin(nullptr);
    if (blockIdx.x == 0 && threadIdx.x == 0 && !p.from) *cleared = 0;
    count[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * (uint32_t)kSortTile, all = p.from ? (uint32_t)__ldcg(p.there) : p.count;
    int2 element[kSortEach];
    sort_elements(p, first + threadIdx.x, kSortThreads, all, element);
#pragma unroll
    for (int k = 0; k < kSortEach; k++)
        if (element[k].x >= 0) atomicAdd(count + sort_digit(p, element[k].x), 1);
    __syncthreads();
    if (threadIdx.x < 1 << p.bits) p.counts[(int64_t)threadIdx.x * p.tiles + blockIdx.x] = count[threadIdx.x];
}
// The sum of the values of the CTA's threads before this one; `sums`: 33 words, whose last one is then the sum of all.
__device__ __forceinline__ int sum_before(int own, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    int run = own;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = run;
    __syncthreads();
    if (warp == 0) {
        const int mine = lane < warps ? sums[lane] : 0;
        int w = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        sums[lane] = w - mine;
        if (lane == 31) sums[32] = w;
    }
    __syncthreads();
    return sums[warp] + run - own;
}
// Of each digit, counts to sums of the tiles before, and the sum of all: a warp a digit.
static __global__ void __launch_bounds__(kSortThreads) pass_sum_kernel(int* counts, int digits, int tiles) {
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, digit = blockIdx.x * kSortWarps + (threadIdx.x >> 5);
    if (digit >= digits) return;
    int* own = counts + (int64_t)digit * tiles;
    int before = 0;
    for (int base = 0; base < tiles; base += 256) {
        int v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = base + 32 * k + lane < tiles ? __ldcg(own + base + 32 * k + lane) : 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            int run = v[k];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += u;
            }
            if (base + 32 * k + lane < tiles) own[base + 32 * k + lane] = before + run - v[k];
            before += __shfl_sync(0xffffffffu, run, 31);
        }
    }
    if (lane == 0) counts[(int64_t)digits * tiles + digit] = before;
}
// An element's rank among its warp's of the same digit, which take EACH x 32 neighbours in order; count: the warp's, of each digit, counted on.
template <int EACH>
__device__ __forceinline__ void warp_ranks(const int (&digit)[EACH], int (&rank)[EACH], int* count) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const unsigned same = __match_any_sync(0xffffffffu, digit[k]);
        rank[k] = digit[k] >= 0 ? count[digit[k]] + __popc(same & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (digit[k] >= 0 && same >> lane == 1u) count[digit[k]] = rank[k] + 1;  // (the last of them)
        __syncwarp();
    }
}
// A warp's elements by their ranks, then the warps before, then the tiles.
static __global__ void __launch_bounds__(kSortThreads) pass_place_kernel(SortPass p) {
    __shared__ int count[kSortWarps][256], sums[33];
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = threadIdx.x; k < kSortWarps * 256; k += kSortThreads) count[k >> 8][k & 255] = 0;
    __syncthreads();
    const uint32_t first = blockIdx.x * (uint32_t)kSortTile + warp * 32 * kSortEach + lane, all = p.from ? (uint32_t)__ldcg(p.there) : p.count;
    int2 element[kSortEach];
    int digit[kSortEach], rank[kSortEach];
    sort_elements(p, first, 32, all, element);
#pragma unroll
    for (int k = 0; k < kSortEach; k++) digit[k] = element[k].x >= 0 ? sort_digit(p, element[k].x) : -1;
    warp_ranks(digit, rank, count[warp]);
    const int digits = 1 << p.bits;
    const int of_digit = threadIdx.x < digits ? __ldcg(p.counts + (int64_t)digits * p.tiles + threadIdx.x) : 0;
    const int before = threadIdx.x < digits ? __ldcg(p.counts + (int64_t)threadIdx.x * p.tiles + blockIdx.x) : 0;
    const int digits_before = sum_before(of_digit, sums);  // (behind its barriers the counts are complete)
    if (!p.from && threadIdx.x == 0 && blockIdx.x == 0) *p.there = sums[32];
    if (threadIdx.x < digits) {
        int at = digits_before + before;
#pragma unroll
        for (int w = 0; w < kSortWarps; w++) {
            const int own = count[w][threadIdx.x];
            count[w][threadIdx.x] = at;
            at += own;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; k++)
        if (digit[k] >= 0) p.to[count[warp][digit[k]] + rank[k]] = element[k];
}

// start[t]: where row t's stretch of the sorted ids begins, t up to n.  What lies between two neighbours, `before` at place i - 1 and `id` at i, is filled in by
// the thread of the second one; where that is much (ids far apart) by its warp, whose places are in a row.
__device__ __forceinline__ void fill_starts(int64_t i, int before, int id, int* start) {
    const int lane = threadIdx.x & 31;
    const int64_t gap = (int64_t)id - before;
    if (gap > 0 && gap <= 32)
        for (int64_t t = before + 1ll; t <= id; t++) start[t] = (int)i;
    for (unsigned wide = __ballot_sync(0xffffffffu, gap > 32); wide; wide &= wide - 1) {
        const int from = __ffs(wide) - 1;
        const int b = __shfl_sync(0xffffffffu, before, from), e = __shfl_sync(0xffffffffu, id, from);
        const int at = (int)(i - lane + from);
        for (int64_t t = b + 1ll + lane; t <= e; t += 32) start[t] = at;
    }
}
constexpr int kStartsEach = 4;
static __global__ void __launch_bounds__(kTableThreads) starts_kernel(const int2* sorted, const int* there, int n, int* start) {
    step_begin(nullptr);
    const int64_t first = (int64_t)blockIdx.x * kTableThreads * kStartsEach + threadIdx.x, count = __ldcg(there);
    int before[kStartsEach], id[kStartsEach];
#pragma unroll
    for (int k = 0; k < kStartsEach; k++) {
        const int64_t i = first + k * kTableThreads;
        before[k] = i == 0 ? -1 : i <= count ? __ldcg(&sorted[i - 1].x) : n, id[k] = i < count ? __ldcg(&sorted[i].x) : n;
    }
#pragma unroll
    for (int k = 0; k < kStartsEach; k++) fill_starts(first + k * kTableThreads, before[k], id[k], start);
}

// A piece of a stretch of more than kLongest: [begin, end) of the sorted ids, and of its row the first piece and how many there are.
struct alignas(16) Piece8 {
    int row, begin, end, first, pieces, rest[3];
};
__device__ __forceinline__ Piece8 load_piece(const Piece8* at) {
    Piece8 p;
    const int4 u = __ldcg(reinterpret_cast<const int4*>(at));
    p.row = u.x, p.begin = u.y, p.end = u.z, p.first = u.w, p.pieces = __ldcg(&at->pieces);
    return p;
}
// count: of long rows' pieces.  They are listed in no order of the rows': it says where a piece's sum is kept, not in which order they are joined.
// A row's pieces are joined kGroup at a time, their sums kGroup at a time, and so on; done[piece][warp's columns] says how many members of a group are there: of a group of
// level l, of kGroup^(l + 1) pieces, at the piece l behind its first one.
constexpr int kLongest = 64, kGroup = 16;
struct Long {
    int* count;
    Piece8* pieces;
    int* done;
    int piece, across;
};
struct Stretch {
    int row, begin, end, pieces, first;
};
__device__ __forceinline__ void list_piece(const Long& l, const Stretch& s, int k) {
    const int begin = s.begin + k * l.piece;
    int4* to = reinterpret_cast<int4*>(l.pieces + s.first + k);
    to[0] = make_int4(s.row, begin, min(begin + l.piece, s.end), s.first);
    to[1] = make_int4(s.pieces, 0, 0, 0);
    if (k % kGroup < 8)
        for (int c = 0; c < l.across; c++) l.done[(int64_t)(s.first + k) * l.across + c] = 0;
}
// Long stretches of more pieces than a lane lists by itself: those for a warp in front, those for all warps behind.
template <int ROOM>
struct ManyPieces {
    Stretch of[ROOM];
    int warps, all;  // how many
    __device__ __forceinline__ void add(const Stretch& s) {
        if (s.pieces > 256)
            of[ROOM - 1 - atomicAdd(&all, 1)] = s;
        else
            of[atomicAdd(&warps, 1)] = s;
    }
    __device__ __forceinline__ void list(const Long& l) const {
        for (int q = (int)threadIdx.x >> 5; q < warps; q += (int)blockDim.x >> 5)
            for (int k = threadIdx.x & 31; k < of[q].pieces; k += 32) list_piece(l, of[q], k);
        for (int q = 0; q < all; q++)
            for (int k = threadIdx.x; k < of[ROOM - 1 - q].pieces; k += (int)blockDim.x) list_piece(l, of[ROOM - 1 - q], k);
    }
};
// A whole warp, a row a lane (from == to: none).
template <int ROOM>
__device__ __forceinline__ void list_long(const Long& l, int t, int from, int to, ManyPieces<ROOM>& many) {
    const int lane = threadIdx.x & 31, own = to - from > kLongest ? (to - from + l.piece - 1) / l.piece : 0;
    if (!__any_sync(0xffffffffu, own > 0)) return;
    int run = own;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
    }
    int base = 0;
    if (lane == 31) base = atomicAdd(l.count, run);
    base = __shfl_sync(0xffffffffu, base, 31);
    const Stretch s{t, from, to, own, base + run - own};
    if (own > 4)
        many.add(s);
    else
        for (int k = 0; k < own; k++) list_piece(l, s, k);
}
static __global__ void __launch_bounds__(kTableThreads) list_long_kernel(const int* start, int n, Long l) {
    __shared__ ManyPieces<kTableThreads> many;
    if (threadIdx.x == 0) many.warps = many.all = 0;
    step_begin(nullptr);
    __syncthreads();
    const int64_t t = (int64_t)blockIdx.x * kTableThreads + threadIdx.x;
    list_long(l, (int)t, t < n ? __ldcg(start + t) : 0, t < n ? __ldcg(start + t + 1) : 0, many);
    __syncthreads();
    many.list(l);
}
// The stretch that begins at place i of `count` sorted ids, id_of(i) each, if it is long: where it ends; else i.
template <class F>
__device__ __forceinline__ int long_end(int i, int count, F id_of) {
    if (i >= count - kLongest) return i;
    const int id = id_of(i);
    if (id_of(i + kLongest) != id || (i > 0 && id_of(i - 1) == id)) return i;
    int in = i + kLongest, out = count;  // places in it, and behind it
    while (out - in > 1) {
        const int between = in + (out - in) / 2;
        (id_of(between) == id ? in : out) = between;
    }
    return out;
}
// ... without starts: a place of the sorted ids a thread
static __global__ void __launch_bounds__(kTableThreads) list_long_places_kernel(const int2* sorted, const int* there, Long l) {
    __shared__ ManyPieces<kTableThreads> many;
    if (threadIdx.x == 0) many.warps = many.all = 0;
    step_begin(nullptr);
    __syncthreads();
    const int count = __ldcg(there), i = (int)(blockIdx.x * kTableThreads + threadIdx.x);
    const int end = long_end(i, count, [&](int at) { return __ldcg(&sorted[at].x); });
    list_long(l, end > i ? __ldcg(&sorted[i].x) : 0, i, end, many);
    __syncthreads();
    many.list(l);
}

// All passes for up to kSortOne ids, the starts (unless that is NULL) and the long stretches: one CTA, the ids in shared memory between the passes.
constexpr int kOneThreads = 1024, kOneEach = 8, kSortOne = kOneThreads * kOneEach;
static __global__ void __launch_bounds__(kOneThreads) sort_one_kernel(SortPass p, int passes, int* start, int* there, Long l) {
    extern __shared__ int2 pairs[];                               // [kSortOne]
    int* const count = reinterpret_cast<int*>(pairs + kSortOne);  // [32][(1 << bits) + 1]
    __shared__ int totals[256], sums[33], pieces;
    __shared__ ManyPieces<kSortOne / kLongest> many;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << p.bits, apart = digits + 1;
    int2 element[kOneEach];
    int digit[kOneEach], rank[kOneEach], all = (int)p.count;
    if (threadIdx.x == 0) pieces = many.warps = many.all = 0;
    sort_elements(p, warp * kOneEach * 32 + lane, 32, p.count, element);
    for (int pass = 0; pass < passes; pass++, p.shift += p.bits) {
        if (pass)
#pragma unroll
            for (int k = 0; k < kOneEach; k++) {
                const int i = (warp * kOneEach + k) * 32 + lane;
                element[k] = i < all ? pairs[i] : make_int2(-1, 0);
            }
        for (int k = threadIdx.x; k < 32 * apart; k += kOneThreads) count[k] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kOneEach; k++) digit[k] = element[k].x >= 0 ? sort_digit(p, element[k].x) : -1;
        warp_ranks(digit, rank, count + warp * apart);
        __syncthreads();
        for (int d = warp; d < digits; d += 32) {  // a lane a warp's count
            const int own = count[lane * apart + d];
            int run = own;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += u;
            }
            count[lane * apart + d] = run - own;
            if (lane == 31) totals[d] = run;
        }
        __syncthreads();
        const int before = sum_before(threadIdx.x < digits ? totals[threadIdx.x] : 0, sums);
        all = sums[32];
        if (threadIdx.x < digits) totals[threadIdx.x] = before;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kOneEach; k++)
            if (digit[k] >= 0) pairs[totals[digit[k]] + count[warp * apart + digit[k]] + rank[k]] = element[k];
        __syncthreads();
    }
    for (int i = threadIdx.x; i < all; i += kOneThreads) p.to[i] = pairs[i];
    if (start)
        for (int i = threadIdx.x; i - lane <= all; i += kOneThreads) {  // (whole warps)
            const int before = i == 0 ? -1 : i <= all ? pairs[i - 1].x : p.n, id = i < all ? pairs[i].x : p.n;
            fill_starts(i, before, id, start);
        }
    if (threadIdx.x == 0) *there = all;
    __syncthreads();
    int* const count_out = l.count;
    l.count = &pieces;
    if (all > kLongest && start)
        for (int t = threadIdx.x; t - lane < p.n; t += kOneThreads) list_long(l, t, t < p.n ? start[t] : 0, t < p.n ? start[t + 1] : 0, many);
    else if (all > kLongest)
        for (int i = threadIdx.x; i - lane < all; i += kOneThreads) {
            const int end = long_end(i, all, [&](int at) { return pairs[at].x; });
            list_long(l, end > i ? pairs[i].x : 0, i, end, many);
        }
    __syncthreads();
    many.list(l);
    if (threadIdx.x == 0) *count_out = pieces;
}

// ---- the gradient

struct TableGrad {
    b200_embed_grad_op a;
    const int2* sorted;
    const int* start;
    const int* there;  // how many sorted ids there are
    Long l;
    float* parts;  // [pieces][ldp]
    int64_t ldp;
    int cuts;      // there may be long stretches
    int vec;       // a row of dtable takes a part's elements together
};
template <class T, int BYTES>
__device__ __forceinline__ void finish_row(const TableGrad& g, int64_t t, int64_t at, float (&sum)[Lanes<T, BYTES>::kEach]) {
#pragma unroll
    for (int k = 0; k < Lanes<T, BYTES>::kEach; k++) sum[k] *= g.a.scale;
    if (g.vec)
        store_sums<T, BYTES, true>(g.a.dtable, t * g.a.lddt, at, g.a.cols, g.a.dtable_type, sum);
    else
        store_sums<T, BYTES, false>(g.a.dtable, t * g.a.lddt, at, g.a.cols, g.a.dtable_type, sum);
}
// n sums, `apart` pieces from one to the next, added up: a row's, or in place of the first of them a group's.  (A call: in line it would take registers from the
// loop that the kernel's time goes to.)
template <class T, int BYTES>
static __device__ __noinline__ void join_pieces(const TableGrad& g, float* parts, int n, int apart, int64_t t, int64_t at) {
    using L = Lanes<T, BYTES>;
    constexpr int kEach = L::kEach, kJoined = kEach > 8 ? 2 : kEach > 4 ? 4 : 8;  // on their way
    float sum[kEach] = {};
    for (int q = 0; q < n; q += kJoined) {
        float v[kJoined][kEach] = {};
#pragma unroll
        for (int i = 0; i < kJoined; i++) {
            const float* row = parts + (int64_t)(q + i) * apart * g.ldp;
            if (q + i >= n) continue;
            if constexpr (BYTES != 0 && L::kOf >= 4) {
#pragma unroll
                for (int k = 0; k < kEach; k += 4)
                    if (L::column(at, k) < g.a.cols) {
                        const float4 f = __ldcg(reinterpret_cast<const float4*>(row + L::column(at, k)));
                        v[i][k] = f.x, v[i][k + 1] = f.y, v[i][k + 2] = f.z, v[i][k + 3] = f.w;
                    }
            } else {
#pragma unroll
                for (int k = 0; k < kEach; k++)
                    if (L::column(at, k) < g.a.cols) v[i][k] = __ldcg(row + L::column(at, k));
            }
        }
#pragma unroll
        for (int i = 0; i < kJoined; i++)
#pragma unroll
            for (int k = 0; k < kEach; k++) sum[k] += v[i][k];
    }
    if (t >= 0)
        finish_row<T, BYTES>(g, t, at, sum);
    else
        store_sums<T, BYTES, true>(parts, 0, at, g.a.cols, B200_TYPE_F32, sum);
}
// Counts this warp in; whether it is the last of n.  What the others wrote before is there then.
__device__ __forceinline__ bool last_of(int* done, int n) {
    __threadfence();
    __syncwarp();
    int before = 0;
    if ((threadIdx.x & 31) == 0) before = atomicAdd(done, 1);
    const bool last = __shfl_sync(0xffffffffu, before, 0) == n - 1;
    if (last) __threadfence();
    return last;
}
// The sum of stretch [from, to) of the sorted ids.
template <class T, int BYTES, int AHEAD>
__device__ __forceinline__ void sum_stretch(const TableGrad& g, int from, int to, int64_t at, float (&sum)[Lanes<T, BYTES>::kEach]) {
    const int lane = threadIdx.x & 31;
    int list = from + lane < to ? __ldcg(&g.sorted[from + lane].y) : 0;
    for (int s = from; s < to; s += 32) {
        const int next = s + 32 + lane < to ? __ldcg(&g.sorted[s + 32 + lane].y) : 0;
        add_first<T, BYTES, AHEAD>(static_cast<const T*>(g.a.dy), g.a.lddy, at, g.a.cols, list, min(32, to - s), sum);
        list = next;
    }
}
// Where the stretch that begins at place `from` ends, or more than kLongest behind it, and its row; `from` itself if none begins there.  A whole warp.
__device__ __forceinline__ int stretch_end(const int2* sorted, int from, int count, int& row) {
    const int lane = threadIdx.x & 31;
    for (int to = from;; to += 31) {  // lane 0: the place before
        const int at = to - 1 + lane, id = at >= 0 && at < count ? __ldcg(&sorted[at].x) : -1;
        const int before = __shfl_sync(0xffffffffu, id, 0);
        if (to == from) {
            row = __shfl_sync(0xffffffffu, id, 1);
            if (before == row) return from;
        }
        const unsigned others = __ballot_sync(0xffffffffu, lane > 0 && id != row);
        if (others) return to + __ffs(others) - 2;
        if (to + 31 - from > kLongest) return to + 31;
    }
}
// Pieces of the long stretches, a warp each, then rows of the table.  Who finishes the last member of a group joins them, in their order.  A CTA's warps count their
// pieces together, behind one fence.  PLACES: there are no starts, and rows without ids are 0 already.  (Asked while it runs, it takes registers: 112 us where 102 had been.)
template <class T, int BYTES, int AHEAD, bool PLACES>
static __global__ void __launch_bounds__(kTableThreads, AHEAD > kGradAhead || BYTES == 0 ? 2 : BYTES == 32 ? 3 : 4) embed_backward_kernel(const __grid_constant__ TableGrad g) {
    using L = Lanes<T, BYTES>;
    constexpr uint32_t kWarps = kTableThreads / 32;
    __shared__ int joins[kWarps];
    step_begin(nullptr);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, across = g.l.across;
    const uint32_t items = g.cuts ? __ldcg(g.l.count) * across : 0;
    for (uint32_t base = blockIdx.x * kWarps; base < items; base += gridDim.x * kWarps) {
        const uint32_t item = base + warp;
        const int64_t at = L::first(item % across);
        if (item < items) {
            const Piece8 piece = load_piece(g.l.pieces + item / across);
            float sum[L::kEach] = {};
            sum_stretch<T, BYTES, AHEAD>(g, piece.begin, piece.end, at, sum);
            store_sums<T, BYTES, true>(g.parts, (int64_t)(item / across) * g.ldp, at, g.a.cols, B200_TYPE_F32, sum);
        }
        __syncthreads();
        if (warp == 0) {
            __threadfence();
            if (lane < kWarps && base + lane < items) {
                const uint32_t row = (base + lane) / across, chunk = (base + lane) % across;
                const Piece8 piece = load_piece(g.l.pieces + row);
                const int group = ((int)row - piece.first) / kGroup * kGroup;
                joins[lane] = atomicAdd(g.l.done + (int64_t)(piece.first + group) * across + chunk, 1) == min(kGroup, piece.pieces - group) - 1;
            }
        }
        __syncthreads();
        if (item < items && joins[warp]) {
            __threadfence();
            const Piece8 piece = load_piece(g.l.pieces + item / across);
            const int n = piece.pieces, own = (int)(item / across) - piece.first;
            for (int apart = 1, level = 1;; apart *= kGroup, level++) {  // of the members of a group, whose first one's place takes their sum
                const int first = own / (apart * kGroup) * (apart * kGroup);
                const bool all = (n - 1) / apart < kGroup;
                join_pieces<T, BYTES>(g, g.parts + (int64_t)(piece.first + first) * g.ldp, min(kGroup, (n - first + apart - 1) / apart), apart, all ? piece.row : -1, at);
                if (all) break;
                const int next = apart * kGroup, next_first = own / next / kGroup * kGroup * next;
                const int members = min(kGroup, (n - next_first + next - 1) / next);
                if (members > 1 && !last_of(g.l.done + (int64_t)(piece.first + next_first + level) * across + item % across, members)) break;
            }
        }
    }
    WarpPlace p((int)across);
    const uint32_t places = PLACES ? (uint32_t)__ldcg(g.there) : (uint32_t)g.a.n;
    for (; p.row < places; p.next()) {
        const int64_t at = L::first(p.at);
        int t = (int)p.row, from = t, to;
        if constexpr (PLACES) {
            to = stretch_end(g.sorted, from, (int)places, t);
            if (to == from) continue;
        } else {
            from = __ldcg(g.start + t), to = __ldcg(g.start + t + 1);
        }
        if (to - from > kLongest) continue;
        float sum[L::kEach] = {};
        sum_stretch<T, BYTES, AHEAD>(g, from, to, at, sum);
        finish_row<T, BYTES>(g, t, at, sum);
    }
}

// ---- the gradient of a table of few rows, as of output buckets: one id a list
//
// HBM bound (131072 x 1024 bf16, 8 rows 56 us, 4.8 TB/s; 262144 x 1024 fp32 180, 6.0), with few lists by latency (5003 x 520 7.7): nothing is sorted.  A warp takes lists
// one after another and the columns that its lanes cover, and keeps a sum for each of the table's rows in shared memory, where each lane meets its own words alone.  A CTA's
// warps are added up in their order, then the CTAs' sums by few_join_kernel.
constexpr int kFewRows = 16, kFewWarps = kTableThreads / 32;
struct FewRows {
    b200_embed_grad_op a;
    float* parts;  // [chunks][across][a CTA's sums, as they lie in shared memory]
    int lists;     // of a warp
    int chunks, across;
};
template <class T, int BYTES>
struct FewSums {
    static constexpr int kEach = Lanes<T, BYTES>::kEach, kVec = kEach < 4 ? kEach : 4, kMany = kEach / kVec;
    static constexpr int kRow = kEach * 32;  // words of a table row's sums
    struct alignas(4 * kVec) Vec {
        float v[kVec];
    };
    // The k-th piece of a lane's sums
    static __device__ __forceinline__ Vec* at(float* sums, int row, int k, int lane) { return reinterpret_cast<Vec*>(sums) + (row * kMany + k) * 32 + lane; }
    // Words 32 row kMany + ..., as at() has them, out to dtable.
    static __device__ __forceinline__ void out(const FewRows& f, int chunk_of_columns, int vec_at, const Vec& v) {
        const int lane = vec_at & 31, k = (vec_at >> 5) % kMany, row = (vec_at >> 5) / kMany;
        const int64_t first = (int64_t)chunk_of_columns * Lanes<T, BYTES>::kWarp + lane * (BYTES ? kEach : 1);
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            const int64_t column = first + (BYTES ? k * kVec + i : 32 * (k * kVec + i));
            if (column < f.a.cols) store_value(f.a.dtable, row * f.a.lddt + column, f.a.dtable_type, v.v[i] * f.a.scale);
        }
    }
};
template <class T, int BYTES>
static __global__ void __launch_bounds__(kTableThreads, 3) few_rows_kernel(const __grid_constant__ FewRows f) {
    using L = Lanes<T, BYTES>;
    using S = FewSums<T, BYTES>;
    constexpr int kAhead = 8;
    extern __shared__ uint4 few_shared[];
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = S::kRow * f.a.n;
    float* const all = reinterpret_cast<float*>(few_shared);
    float* const sums = all + warp * part;
    const uint32_t chunk = blockIdx.x / (uint32_t)f.across, columns = blockIdx.x % (uint32_t)f.across;
    for (int k = lane; k < part; k += 32) sums[k] = 0.f;
    __syncwarp();
    const int64_t at = L::first(columns), first = ((int64_t)chunk * kFewWarps + warp) * f.lists, last = min(first + f.lists, (int64_t)f.a.rows);
    const T* dy = static_cast<const T*>(f.a.dy);
    int64_t id = first + lane < last ? id_at(f.a.ids, (first + lane) * f.a.ldids, f.a.wide_ids, f.a.n) : -1;
    for (int64_t s = first; s < last; s += 32) {
        const int64_t next = s + 32 + lane < last ? id_at(f.a.ids, (s + 32 + lane) * f.a.ldids, f.a.wide_ids, f.a.n) : -1;
        for (unsigned mask = __ballot_sync(0xffffffffu, id >= 0); mask;) {
            L row[kAhead];
            int to[kAhead];
            const int there = min(kAhead, __popc(mask));
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int from = __ffs(mask) - 1;  // (0 left: not used)
                mask &= mask - 1;
                to[k] = __shfl_sync(0xffffffffu, (int)id, from);
                if (k < there) row[k].load(dy + (s + from) * f.a.lddy, at, f.a.cols);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (k >= there) continue;
                float sum[L::kEach];
#pragma unroll
                for (int q = 0; q < S::kMany; q++) {
                    const typename S::Vec v = *S::at(sums, to[k], q, lane);
#pragma unroll
                    for (int i = 0; i < S::kVec; i++) sum[q * S::kVec + i] = v.v[i];
                }
                row[k].add(sum);
#pragma unroll
                for (int q = 0; q < S::kMany; q++) {
                    typename S::Vec v;
#pragma unroll
                    for (int i = 0; i < S::kVec; i++) v.v[i] = sum[q * S::kVec + i];
                    *S::at(sums, to[k], q, lane) = v;
                }
            }
        }
        id = next;
    }
    __syncthreads();
    using Vec = typename S::Vec;
    const int vecs = part / S::kVec;
    for (int k = threadIdx.x; k < vecs; k += kTableThreads) {
        Vec sum = reinterpret_cast<const Vec*>(all)[k];
#pragma unroll
        for (int w = 1; w < kFewWarps; w++) {
            const Vec v = reinterpret_cast<const Vec*>(all + w * part)[k];
#pragma unroll
            for (int i = 0; i < S::kVec; i++) sum.v[i] += v.v[i];
        }
        if (f.chunks == 1)
            S::out(f, (int)columns, k, sum);
        else
            reinterpret_cast<Vec*>(f.parts + (int64_t)blockIdx.x * part)[k] = sum;
    }
}
// The CTAs' sums: 32 pieces of a chunk of columns a CTA, whose warps take every eighth of the parts.
template <class T, int BYTES>
static __global__ void __launch_bounds__(kTableThreads) few_join_kernel(const __grid_constant__ FewRows f) {
    using S = FewSums<T, BYTES>;
    using Vec = typename S::Vec;
    __shared__ Vec shared[kFewWarps][32];
    step_begin(nullptr);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = S::kMany * f.a.n;  // (of 32 pieces)
    const int columns = blockIdx.x / rows, at = blockIdx.x % rows * 32 + lane;
    const float* const parts = f.parts + (int64_t)columns * S::kRow * f.a.n;
    Vec sum{};
#pragma unroll 8
    for (int c = warp; c < f.chunks; c += kFewWarps) {
        const float* from = parts + (int64_t)c * f.across * S::kRow * f.a.n + at * S::kVec;
        Vec v;
        if constexpr (S::kVec == 4) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(from));
            v.v[0] = w.x, v.v[1] = w.y, v.v[2] = w.z, v.v[3] = w.w;
        } else {
#pragma unroll
            for (int i = 0; i < S::kVec; i++) v.v[i] = __ldcg(from + i);
        }
#pragma unroll
        for (int i = 0; i < S::kVec; i++) sum.v[i] += v.v[i];
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < kFewWarps; w++)
#pragma unroll
        for (int i = 0; i < S::kVec; i++) sum.v[i] += shared[w][lane].v[i];
    S::out(f, columns, at, sum);
}

}  // namespace b200
