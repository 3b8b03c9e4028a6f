// Products of matrices in 4 bits on the tensor pipe, for the dense trunk's layers.
//
//   d[m][n] = act(sum over k of a(m, k) b(n, k) + bias[n]) + residual[m][n]
//
// a: rows of codes along k, b: a row of codes per output, each with a power of two for every 32 of k (kernels_four.cuh).  The tensor pipe
// multiplies codes and scales as they are (tcgen05.mma.kind::mxf4.block_scale): nothing is turned into wider types.
//
// As product_kernel (kernels_product.cuh): CTAs, or pairs of them, take tiles one after another; one thread has TMA fetch stages of 128 bytes of
// k = 256 codes, 128-byte swizzled; one warp issues the products; eight or sixteen take finished sums out, 32 columns at a time, and hand them to TMA in boxes
// of 32 rows of 64 bytes.  (Eight warps for a tile of 256 columns, 64 at a time: 7000 clocks a tile, most of them spent fetching instructions.)
// Sums stay in tensor memory over all of k: the pipe cuts a sum off at each of its k / 64 additions, by 2^-24 of it or so.
//
// Scales have to lie in tensor memory.  They come with the stages, and four more warps, one for each 32 lanes, carry them on through registers.  The pipe's own
// copies from shared memory (tcgen05.cp, 512 bytes each) take it 100 clocks a piece, in which it multiplies nothing: six of them 330 ns of a stage's 800, where
// its four products of 256 x 256 x 64 are 280 and a stage is now 290.  (Loaded from global memory by those warps: 1500, as each arrival at a barrier
// waited for the loads on their way.)
// Two tiles' sums of 256 columns and the scales of five stages do not fit in 512 columns: the tiles overlap by half, which is taken out first.
// (Scales of two stages, and an overlap of 64 columns: the way from the products that last used a place, by way of those warps, to those that use it
// next is longer than one stage's products: 1050 ns a stage.)
//
// Measured, us: 131072 x 2048 -> 512 71 (3.9 PFLOP/s, under the power cap: 64 with codes of zeros; a tile's eight stages 2.3 us, 0.95 until the next one's begin, 3.6
// together; HBM 42); 16384 x 1024 -> 2048 23, with SCReLU 25, with a residual 33.
#pragma once
#include "kernels_four.cuh"
#include "product_out.cuh"

namespace b200 {

template <int BN, bool PAIR, bool ADDS>
struct Tile4 {
    static constexpr int kRows = PAIR ? 256 : 128, kOwnColumns = PAIR ? BN / 2 : BN;  // of b, that this CTA fetches
    static constexpr int kScaleTiles = (BN + 127) / 128;                              // of b's rows: each CTA of a pair wants all of them
    static constexpr uint32_t kA = 128 * 128, kB = kOwnColumns * 128, kAScales = 1024, kScales = kAScales * (1 + kScaleTiles), kStage = kA + kB + kScales;
    static constexpr int kTakers = BN / 16, kGroups = kTakers / 4;  // warps that take sums out: a quarter of the rows, 32 columns of every 32 kGroups
    static constexpr int kThreads = 64 + 32 * kTakers + 128;
    static constexpr uint32_t kBox = 32 * 64;
    static constexpr size_t kBoxes = kTakers * kBox * (ADDS ? 2 : 1), kValues = (size_t)kTakers * 64 * 4, kRest = 1024 + kBoxes + kValues;
    static constexpr int kFit = (int)((232448 - 1024 - kRest) / kStage), kStages = kFit < 8 ? kFit : 8;
    static constexpr size_t kShared = kRest + (size_t)kStages * kStage;
    static constexpr int kScaleWords = 2 * 4 * (1 + kScaleTiles);              // columns of tensor memory for a stage's: a's of two tiles of k, b's
    static constexpr int kSumsApart = 128;                                     // of two tiles: those of 256 columns share half of their places
    static constexpr bool kShares = BN > kSumsApart;
    static constexpr uint32_t kScalesAt = kSumsApart + BN;
    static_assert(kScalesAt + kStages * kScaleWords <= 512 && kStages >= 3, "");
    static_assert(2 * 32 * kGroups == BN && (!kShares || 32 * kGroups == kSumsApart), "a warp takes 32 columns twice, those of shared places together");
};

// A row of 64 bytes of a box, the residual there added, in place: v from `from` on, 32 values of 16 bits or 16 of fp32.  64-byte swizzle; r: the row's number.
template <class T>
__device__ __forceinline__ void box_out64(unsigned char* row, int r, const float (&v)[32], int from, bool residual) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        uint4* at = reinterpret_cast<uint4*>(row + ((k ^ (r >> 1 & 3)) << 4));
        constexpr int kEach = 16 / sizeof(T);
        float x[kEach];
#pragma unroll
        for (int q = 0; q < kEach; q++) x[q] = v[from + kEach * k + q];
        if (residual) {
            const uint4 o = *at;
            const uint32_t u[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if constexpr (sizeof(T) == 4) {
                    x[q] += __uint_as_float(u[q]);
                } else {
                    float low, high;
                    unpack2<T>(u[q], low, high);
                    x[2 * q] += low, x[2 * q + 1] += high;
                }
            }
        }
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if constexpr (sizeof(T) == 4)
                w[q] = __float_as_uint(x[q]);
            else
                w[q] = pack2<T>(x[2 * q], x[2 * q + 1]);
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// Sixteen columns of a box of fp32, the residual added, element by element: half a warp a row.
template <class T>
static __device__ __forceinline__ void columns_out16(const ProductArgs& p, const unsigned char* box, int lane, int64_t rows0, int64_t column0, bool adds) {
    const int64_t column = column0 + (lane & 15);
    if (column >= p.n) return;
#pragma unroll 4
    for (int k = 0; k < 16; k++) {
        const int r = 2 * k + (lane >> 4);
        const int64_t row = rows0 + r;
        if (row >= p.m) break;
        float x = *reinterpret_cast<const float*>(box + r * 64 + (((lane >> 2 & 3) ^ (r >> 1 & 3)) << 4) + (lane & 3) * 4);
        if (adds) x += to_float(static_cast<const T*>(p.residual)[row * p.ldr + column]);
        static_cast<T*>(p.d)[row * p.ldd + column] = from_float<T>(x);
    }
}
// Four columns of a warp's 32 lanes into tensor memory.  What was put is there behind scales_stored().
__device__ __forceinline__ void put_scales(uint32_t to, const uint4& w) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
}
__device__ __forceinline__ void scales_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// An arrival that says nothing of memory but tensor memory, whose instructions the fence in front of it orders.  (One that releases waits for all else that
// the warp has had to do with memory: 1500 clocks between the scales' stores and those who wait for them.)
__device__ __forceinline__ void arrive_for_tensor_memory(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Form of a product of e2m1 with exponents as scales: `half` says which two bytes of a word of scales belong to its 64 of k.
__device__ __forceinline__ uint32_t four_form(int m, int n, uint32_t half) {
    return half << 5 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(m >> 4) << 24 | half << 30;
}
// One of the warp's lanes, the same one every time.
__device__ __forceinline__ bool elected() {
    uint32_t is;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(is));
    return is != 0;
}
// a, b: where the tiles lie in shared memory, in pieces of 16 bytes
template <bool PAIR>
__device__ __forceinline__ void multiply4(uint32_t sums, uint32_t a, uint32_t b, uint32_t form, uint32_t a_scales, uint32_t b_scales, bool add) {
    // (tile_descriptor's: rows of 128 bytes along k, 128-byte swizzle)
#define B200_MULTIPLY4(group)                                                                                                                                                   \
    asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %7};\nmov.b64 b, {%2, %7};\ntcgen05.mma.cta_group::" group                           \
                 ".kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%5], [%6], p;\n}" ::"r"(sums),                                                                         \
                 "r"((a & 0x3fffu) | 1u << 16), "r"((b & 0x3fffu) | 1u << 16), "r"(form), "r"((int)add), "r"(a_scales), "r"(b_scales), "r"(64u | 1u << 14 | 2u << 29)             \
                 : "memory")
    if constexpr (PAIR)
        B200_MULTIPLY4("2");
    else
        B200_MULTIPLY4("1");
#undef B200_MULTIPLY4
}

// The tiles that a CTA or a pair takes, one after another, and where they lie; no division behind the first one's.
struct TileAt {
    uint32_t tile, row, column, step, rows_on, columns_on, across;
    __device__ __forceinline__ TileAt(uint32_t first, uint32_t step_, uint32_t across_)
        : tile(first), row(first / across_), column(first % across_), step(step_), rows_on(step_ / across_), columns_on(step_ % across_), across(across_) {}
    __device__ __forceinline__ void next() {
        tile += step, row += rows_on, column += columns_on;
        if (column >= across) column -= across, row++;
    }
};

template <int BN, bool PAIR, bool ADDS>
static __global__ void __launch_bounds__((Tile4<BN, PAIR, ADDS>::kThreads), 1)
    product4_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ CUtensorMap a_scale_map,
                    const __grid_constant__ CUtensorMap b_scale_map, const __grid_constant__ CUtensorMap d_map, const __grid_constant__ CUtensorMap r_map, const ProductArgs p) {
    using T = Tile4<BN, PAIR, ADDS>;
    constexpr int kStages = T::kStages, kCtas = PAIR ? 2 : 1;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t full[kStages], empty[kStages], scales_in[kStages], sums_done[2], sums_free[2], residual_in[2 * T::kTakers];
    __shared__ uint32_t memory_at;
    __shared__ int dead;
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const WaitsFor<false> wait{&dead, p.gave_up};
    if (threadIdx.x == 0) {
        dead = 0;
        for (int s = 0; s < kStages; s++) {
            mbar_init(&full[s], 1 + 4 * kCtas);  // (the codes, and each warp that carries scales on)
            mbar_init(&empty[s], 1);
            mbar_init(&scales_in[s], 1);
        }
        for (int k = 0; k < 2 * T::kTakers; k++) mbar_init(&residual_in[k], 1);
        for (int k = 0; k < 2; k++) {
            mbar_init(&sums_done[k], 1);
            mbar_init(&sums_free[k], T::kTakers * kCtas);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (threadIdx.x == 32) {
        know_map(&a_map);
        know_map(&b_map);
        know_map(&a_scale_map);
        know_map(&b_scale_map);
        if (p.boxes) know_map(&d_map);
    }
    __syncwarp();
    if (warp == 1) tensor_memory_take<PAIR>(&memory_at, 512);
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tensor_fence_after();
    const uint32_t memory = memory_at;

    const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n;
    const TileAt start(blockIdx.x / kCtas, gridDim.x / kCtas, (uint32_t)p.tiles_n);
    if (warp == 0) {
        if (lane == 0) {  // fetches
            int s = 0;
            uint32_t phase = 1;  // (a new barrier's phase before is over)
            for (TileAt at = start; at.tile < tiles && !dead; at.next()) {
                const int m0 = (int)(at.row * T::kRows + 128 * rank), n0 = (int)(at.column * BN);
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    if (!wait(&empty[s], phase)) break;
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA;
                    const uint32_t bar = PAIR ? of_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
                    if (rank == 0) mbar_expect_tx(&full[s], kCtas * (T::kA + T::kB));
                    mbar_expect_tx(&scales_in[s], T::kScales);
                    load_box3(b_at + T::kB, &a_scale_map, 0, 2 * kb, m0 >> 7, smem_u32(&scales_in[s]));
                    load_box3(b_at + T::kB + T::kAScales, &b_scale_map, 0, 2 * kb, n0 >> 7, smem_u32(&scales_in[s]));
                    load_box<PAIR>(a_at, &a_map, kb * 128, m0, bar);
                    load_box<PAIR>(b_at, &b_map, kb * 128, n0 + (PAIR ? T::kOwnColumns * (int)rank : 0), bar);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {  // multiplies: the whole warp keeps count, one lane issues (operands that all lanes agree on need no way into uniform registers)
            // The pair's other CTA arrives at these barriers too, whose tensor memory the products read and write.  (The other waits are for this CTA's own copies and
            // for what the tensor pipe leaves; at the pair's scope they take 16384 x 1024 -> 2048 26.1 us instead of 25.4, these alone nothing.)
            const WaitsFor<PAIR> wait{&dead, p.gave_up};
            const bool issues = elected();
            const uint32_t a0 = smem_u32(base) >> 4, form = four_form(T::kRows, BN, 0), other = four_form(T::kRows, BN, 1);
            const int whole = (int)(p.k / 256), rest = (int)((p.k % 256 + 63) / 64);  // stages, and products of the last one (past k there may be no scales)
            int s = 0;
            uint32_t phase = 0, done = 0;
            bool fine = true;  // (of all lanes: they leave together)
            for (TileAt at = start; at.tile < tiles && fine; at.next(), done++) {
                const uint32_t half = done & 1, sums = memory + half * T::kSumsApart;
                fine = __all_sync(0xffffffffu, T::kShares ? done == 0 || wait(&sums_free[0], done - 1 & 1) : wait(&sums_free[half], (done >> 1 & 1) ^ 1));
                if (!fine) break;
                tensor_fence_after();
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    fine = __all_sync(0xffffffffu, wait(&full[s], phase));
                    if (!fine) break;
                    tensor_fence_after();
                    const uint32_t a_at = a0 + s * (T::kStage / 16), b_at = a_at + T::kA / 16, a_scales = memory + T::kScalesAt + s * T::kScaleWords, b_scales = a_scales + 8;
                    if (issues) {
                        auto product = [&](int q) {
                            const uint32_t g = q >> 1, part = (uint32_t)(q & 1) << 31;
                            multiply4<PAIR>(sums, a_at + 2 * q, b_at + 2 * q, q & 1 ? other : form, a_scales + 4 * g + part, b_scales + 4 * T::kScaleTiles * g + part, kb > 0 || q > 0);
                        };
                        if (kb < whole) {
#pragma unroll
                            for (int q = 0; q < 4; q++) product(q);
                        } else {
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                if (q < rest) product(q);
                        }
                        when_multiplied<PAIR>(&empty[s]);
                        if (kb + 1 == p.k_blocks) when_multiplied<PAIR>(&sums_done[half]);
                    }
                    __syncwarp();
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp < 2 + T::kTakers) {  // takes sums out: 32 rows, twice 32 columns
        constexpr int kApart = 32 * T::kGroups;
        const int quarter = warp & 3, taker = warp - 2, c0 = taker / 4 * 32;
        unsigned char* const boxes = base + kStages * T::kStage + taker * T::kBox * (ADDS ? 2 : 1);
        float* bias = reinterpret_cast<float*>(base + kStages * T::kStage + T::kBoxes) + taker * 64;
        const bool wide = p.d_type == B200_TYPE_F32;
        int64_t bias_at = -1;
        // Where the boxes lie, in their order: of two tiles that share places the second half of the one, and the first half of the other, first; fp32, and what
        // is written element by element, 16 columns a box.
        struct Where {
            TileAt at;
            uint32_t done;
            int k, h;
        };
        auto column_of = [&](uint32_t done, int k) { return (kApart * k + (T::kShares && (done & 1) == 0 ? kApart : 0)) % BN; };  // of the tile, behind c0
        auto first_row = [&](const TileAt& at) { return (int64_t)at.row * T::kRows + 128 * rank + 32 * quarter; };
        auto first_column = [&](const Where& w) { return (int64_t)w.at.column * BN + c0 + column_of(w.done, w.k) + 16 * w.h; };
        // ADDS and boxes: a box's residual is on its way while the box before it is filled.  (Loaded into registers, 64 bytes of a lane's row, it takes
        // twice the time: 16384 x 1024 -> 2048 37 us so when tried, 71 in registers, 41 with one box.)
        Where next{start, 0, 0, 0};
        uint32_t filled = 0;  // boxes
        auto fetch_residual = [&](uint32_t number) {
            auto on = [&] {
                next.h = wide && next.h == 0;
                if (next.h == 0 && (next.k ^= 1) == 0) next.at.next(), next.done++;
            };
            while (next.at.tile < tiles && (first_row(next.at) >= p.m || first_column(next) >= p.n)) on();
            if (next.at.tile >= tiles) return;
            if (lane == 0) {
                bulk_wait_read<0>();
                uint64_t* bar = &residual_in[2 * taker + (number & 1)];
                mbar_expect_tx(bar, T::kBox);
                load_box3(smem_u32(boxes + (number & 1) * T::kBox), &r_map, (int)first_column(next), (int)first_row(next.at), 0, smem_u32(bar));
            }
            on();
        };
        const bool ahead = ADDS && p.boxes;
        if (ahead) fetch_residual(0);
        uint32_t done = 0;
        bool fine = true;
        for (TileAt at = start; at.tile < tiles && fine; at.next(), done++) {
            const int half = done & 1;
            const int64_t rows0 = first_row(at), own0 = (int64_t)at.column * BN + c0;
            const int own = rows0 < p.m ? (int)min((int64_t)BN, p.n - own0) : 0;  // columns there are from own0 on, 0 or less: nothing here
            if (bias_at != own0) {
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 2; k++) bias[32 * k + lane] = p.bias && kApart * k + lane < own ? __ldg(p.bias + own0 + kApart * k + lane) : 0.f;
                bias_at = own > 0 ? own0 : -1;  // (rows past the last: nothing was loaded)
                __syncwarp();
            }
            fine = __all_sync(0xffffffffu, wait(&sums_done[half], done >> 1 & 1));
            if (!fine) break;
            tensor_fence_after();
            const uint32_t sums = memory + ((uint32_t)quarter << 21) + half * T::kSumsApart + c0;
#pragma unroll 1
            for (int k = 0; k < 2; k++) {
                const int c1 = column_of(done, k);
                float v[32];
                if (c1 < own) load_sums32(sums + c1, v);
                if (k == (T::kShares ? 0 : 1)) {  // the next tile, once the places that it shares are read (or all); every warp has read the tile before
                    tensor_fence_before();
                    __syncwarp();
                    uint64_t* bar = &sums_free[T::kShares ? 0 : half];
                    if (lane == 0) arrive_for_tensor_memory(PAIR ? of_rank(smem_u32(bar), 0) : smem_u32(bar));
                }
                if (c1 >= own) continue;
                finish_sums<false, true>(p, v, 1.f, bias + (c1 ? 32 : 0), nullptr, true);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int c = c1 + 16 * h;
                    if (h && ((p.boxes && !wide) || c >= own)) break;
                    unsigned char* box = boxes + (ahead ? (filled & 1) * T::kBox : 0);
                    unsigned char* row = box + lane * 64;
                    if (ahead) {
                        fetch_residual(filled + 1);
                        fine = __all_sync(0xffffffffu, wait(&residual_in[2 * taker + (filled & 1)], filled >> 1 & 1));
                        if (!fine) break;
                        filled++;
                    } else if (p.boxes) {
                        if (lane == 0) bulk_wait_read<0>();
                        __syncwarp();
                    }
                    if (!p.boxes)
                        box_out64<float>(row, lane, v, 16 * h, false);
                    else if (wide)
                        box_out64<float>(row, lane, v, 16 * h, ADDS);
                    else if (p.d_type == B200_TYPE_BF16)
                        box_out64<bf16>(row, lane, v, 0, ADDS);
                    else
                        box_out64<f16>(row, lane, v, 0, ADDS);
                    if (p.boxes) {
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            store_box3(&d_map, smem_u32(box), (int)own0 + c, (int)rows0, 0);
                            bulk_commit();
                        }
                        __syncwarp();
                    } else {
                        __syncwarp();
                        if (wide)
                            columns_out16<float>(p, box, lane, rows0, own0 + c, ADDS);
                        else if (p.d_type == B200_TYPE_BF16)
                            columns_out16<bf16>(p, box, lane, rows0, own0 + c, ADDS);
                        else
                            columns_out16<f16>(p, box, lane, rows0, own0 + c, ADDS);
                        __syncwarp();
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_all();
    } else {  // carries scales on, 32 lanes of them
        const uint32_t to = memory + ((uint32_t)(warp & 3) << 21) + T::kScalesAt;
        int s = 0;
        uint32_t phase = 0;
        bool fine = true;
        for (TileAt at = start; at.tile < tiles && fine; at.next()) {
            for (int kb = 0; kb < p.k_blocks; kb++) {
                // (they were fetched behind the products that last used this place, here and in tensor memory)
                fine = __all_sync(0xffffffffu, wait(&scales_in[s], phase));
                if (!fine) break;
                tensor_fence_after();
                // tiles of a's scales for 128 of k each, then for each 128 of k those of b
                const uint4* from = reinterpret_cast<const uint4*>(base + s * T::kStage + T::kA + T::kB) + lane;
                uint4 w[T::kScaleWords / 4];
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    w[g] = from[32 * g];
#pragma unroll
                    for (int t = 0; t < T::kScaleTiles; t++) w[2 + T::kScaleTiles * g + t] = from[(T::kAScales + 1024 * t + 512 * g) / 16];
                }
#pragma unroll
                for (int k = 0; k < T::kScaleWords / 4; k++) put_scales(to + s * T::kScaleWords + 4 * k, w[k]);
                scales_stored();
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) arrive_for_tensor_memory(PAIR ? of_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]));
                if (++s == kStages) s = 0, phase ^= 1;
            }
        }
    }
    __syncwarp();
    if (dead) {  // what is in flight lands before the CTA's memory goes
        for (int k = 0; k < 2000; k++) __nanosleep(1000);
    }
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    if (warp == 1) {
        tensor_fence_after();
        tensor_memory_give<PAIR>(memory, 512);
    }
}

}  // namespace b200
