// Products of matrices in 4 bits on the tensor pipe, for the dense trunk's layers.
//
//   d[m][n] = act(sum over k of a(m, k) b(n, k) + bias[n]) + residual[m][n]
//
// a: rows of codes along k, b: a row of codes per output, each with a power of two for every 32 of k (kernels_four.cuh).  The tensor pipe
// multiplies codes and scales as they are (tcgen05.mma.kind::mxf4.block_scale): nothing is turned into wider types.
//
// As product_kernel (kernels_product.cuh): CTAs, or pairs of them, take tiles one after another; one thread has TMA fetch stages of 128 bytes of
// k = 256 codes, 128-byte swizzled, and their scales' tiles; one copies the scales on into tensor memory and issues the products; eight warps
// take finished sums out and hand them to TMA in boxes of 32 rows of 128 bytes.
// Sums stay in tensor memory over all of k: the pipe cuts a sum off at each of its k / 64 additions, by 2^-24 of it or so.
#pragma once
#include "kernels_four.cuh"
#include "product_out.cuh"

namespace b200 {

template <int BN, bool PAIR>
struct Tile4 {
    static constexpr int kRows = PAIR ? 256 : 128, kOwnColumns = PAIR ? BN / 2 : BN;  // of b, that this CTA fetches
    static constexpr int kCodes = 256;                                                // of k in a stage: 128 bytes
    static constexpr uint32_t kA = 128 * 128, kB = kOwnColumns * 128;
    static constexpr int kScaleTiles = (BN + 127) / 128;  // of b's rows: each CTA of a pair wants all of them
    static constexpr uint32_t kAScales = 1024, kBScales = kScaleTiles * 1024, kStage = kA + kB + kAScales + kBScales;
    static constexpr int kTakers = 8, kOwn = BN * 4 / kTakers;  // warps that take sums out, columns of each
    static constexpr int kThreads = 64 + 32 * kTakers;
    static constexpr size_t kBoxes = kTakers * 4096, kValues = (size_t)kTakers * kOwn * 4, kRest = 1024 + kBoxes + kValues;
    static constexpr int kFit = (int)((232448 - 1024 - kRest) / kStage), kStages = kFit < 8 ? kFit : 8;
    static constexpr size_t kShared = kRest + (size_t)kStages * kStage;
    static constexpr int kSums = BN == 256 ? 1 : 2;                          // tiles whose sums there is room for
    static constexpr uint32_t kScaleColumns = 2 * (4 + 4 * kScaleTiles);     // of tensor memory for a stage's scales
    static constexpr uint32_t kScalesAt = 512 - 2 * kScaleColumns;           // two stages' by turns
    static_assert(kSums * BN <= kScalesAt && kStages >= 3, "");
    static_assert(kStage % 1024 == 0, "the swizzle wants stages on 1024 bytes");
};

// A box of a stack of scales' tiles into shared memory; the bytes are counted at `bar`, of this CTA or (PAIR) of either.
template <bool PAIR>
__device__ __forceinline__ void load_scales(uint32_t to, const CUtensorMap* map, int y, int z, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to), "l"(map), "r"(0),
                     "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else
        load_box3(to, map, 0, y, z, bar);
}
// A tile of scales, 32 rows of 16 bytes, from shared memory into four columns of tensor memory, once for each of its four parts of 32 lanes (PAIR: of
// both CTAs, from and to the same places of each).
template <bool PAIR>
__device__ __forceinline__ void scales_on(uint32_t to, uint32_t smem) {
    const uint64_t from = (uint64_t)((smem & 0x3ffffu) >> 4) | (uint64_t)(128u >> 4 | 1u << 14) << 32;  // (eight rows are 128 bytes, no swizzle)
    if constexpr (PAIR)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from) : "memory");
}
// Form of a product of e2m1 with exponents as scales: `half` says which two bytes of a word of scales belong to its 64 of k.
__device__ __forceinline__ uint32_t four_form(int m, int n, uint32_t half) {
    return half << 5 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(m >> 4) << 24 | half << 30;
}
template <bool PAIR>
__device__ __forceinline__ void multiply4(uint32_t sums, uint64_t a, uint64_t b, uint32_t form, uint32_t a_scales, uint32_t b_scales, bool add) {
#define B200_MULTIPLY4(group)                                                                                                                       \
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::" group ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n}" ::"r"( \
                     sums),                                                                                                                         \
                 "l"(a), "l"(b), "r"(form), "r"((int)add), "r"(a_scales), "r"(b_scales)                                                             \
                 : "memory")
    if constexpr (PAIR)
        B200_MULTIPLY4("2");
    else
        B200_MULTIPLY4("1");
#undef B200_MULTIPLY4
}

template <int BN, bool PAIR>
static __global__ void __launch_bounds__((Tile4<BN, PAIR>::kThreads), 1)
    product4_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ CUtensorMap a_scale_map,
                    const __grid_constant__ CUtensorMap b_scale_map, const __grid_constant__ CUtensorMap d_map, const __grid_constant__ CUtensorMap r_map, const ProductArgs p) {
    using T = Tile4<BN, PAIR>;
    constexpr int kStages = T::kStages, kCtas = PAIR ? 2 : 1;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t full[kStages], empty[kStages], sums_done[2], sums_free[2], residual_in[T::kTakers];
    __shared__ uint32_t memory_at;
    __shared__ int dead;
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const Waits wait{&dead, p.gave_up};
    if (threadIdx.x == 0) {
        dead = 0;
        for (int s = 0; s < kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int k = 0; k < T::kTakers; k++) mbar_init(&residual_in[k], 1);
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

    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    const int64_t first = blockIdx.x / kCtas, step = gridDim.x / kCtas;
    if (warp == 0) {
        if (lane == 0) {  // fetches
            int s = 0;
            uint32_t phase = 1;  // (a new barrier's phase before is over)
            for (int64_t tile = first; tile < tiles && !dead; tile += step) {
                const int m0 = (int)(tile / p.tiles_n * T::kRows) + 128 * (int)rank, n0 = (int)(tile % p.tiles_n * BN);
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    if (!wait(&empty[s], phase)) break;
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA, scales_at = b_at + T::kB;
                    const uint32_t bar = PAIR ? of_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
                    if (rank == 0) mbar_expect_tx(&full[s], kCtas * T::kStage);
                    load_box<PAIR>(a_at, &a_map, kb * 128, m0, bar);
                    load_box<PAIR>(b_at, &b_map, kb * 128, n0 + (PAIR ? T::kOwnColumns * (int)rank : 0), bar);
                    load_scales<PAIR>(scales_at, &a_scale_map, 2 * kb, m0 >> 7, bar);
                    load_scales<PAIR>(scales_at + T::kAScales, &b_scale_map, 2 * kb, n0 >> 7, bar);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {  // multiplies
            int s = 0, done = 0;
            uint32_t phase = 0, turn = 0;
            for (int64_t tile = first; tile < tiles && !dead; tile += step, done++) {
                const int half = done % T::kSums;
                const uint32_t sums = memory + half * BN;
                bool fine = wait(&sums_free[half], (done / T::kSums & 1) ^ 1);
                if (!fine) break;
                tensor_fence_after();
                for (int kb = 0; kb < p.k_blocks; kb++) {
                    fine = wait(&full[s], phase);
                    if (!fine) break;
                    tensor_fence_after();
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA, scales_at = b_at + T::kB;
                    const int quarters = (int)min((int64_t)4, (p.k - (int64_t)kb * 256 + 63) / 64);  // (past k there may be no scales)
                    // (the products before the last ones with these columns are done with them: the pipe takes copies and products in order)
                    const uint32_t a_scales = memory + T::kScalesAt + turn * T::kScaleColumns, b_scales = a_scales + 8;
                    turn ^= 1;
                    for (int g = 0; 2 * g < quarters; g++) {
                        scales_on<PAIR>(a_scales + 4 * g, scales_at + 512 * g);
#pragma unroll
                        for (int t = 0; t < T::kScaleTiles; t++)
                            scales_on<PAIR>(b_scales + 4 * T::kScaleTiles * g + 4 * t, scales_at + T::kAScales + 1024 * t + 512 * g);
                    }
                    for (int q = 0; q < quarters; q++) {
                        const uint32_t part = (uint32_t)(q & 1), g = (uint32_t)q >> 1;
                        multiply4<PAIR>(sums, tile_descriptor(a_at + q * 32, 16), tile_descriptor(b_at + q * 32, 16), four_form(T::kRows, BN, part),
                                        a_scales + 4 * g + (part << 31), b_scales + 4 * T::kScaleTiles * g + (part << 31), kb > 0 || q > 0);
                    }
                    when_multiplied<PAIR>(&empty[s]);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                when_multiplied<PAIR>(&sums_done[half]);
            }
        }
    } else {  // takes sums out, kOwn columns of 32 rows
        const int quarter = warp & 3, taker = warp - 2, c0 = taker / 4 * T::kOwn;
        unsigned char* box = base + kStages * T::kStage + taker * 4096;
        float* bias = reinterpret_cast<float*>(base + kStages * T::kStage + T::kBoxes) + taker * T::kOwn;
        const bool wide = p.boxes && p.d_type == B200_TYPE_F32, adds = p.residual;
        const int width = wide ? 32 : 64;  // columns of a box
        uint32_t residuals = 0;
        int done = 0;
        for (int64_t tile = first; tile < tiles; tile += step, done++) {
            const int64_t rows0 = tile / p.tiles_n * T::kRows + 128 * rank + 32 * quarter, own0 = tile % p.tiles_n * BN + c0;
            const int own = rows0 < p.m ? (int)min((int64_t)T::kOwn, p.n - own0) : 0;  // columns there are, 0 or less: nothing here
            auto fetch_residual = [&](int c) {
                if (lane == 0) {
                    bulk_wait_read<0>();
                    mbar_expect_tx(&residual_in[taker], 4096);
                    load_box3(smem_u32(box), &r_map, (int)own0 + c, (int)rows0, 0, smem_u32(&residual_in[taker]));
                }
            };
            if (adds && p.boxes && own > 0) fetch_residual(0);
            __syncwarp();
            for (int c = lane; c < T::kOwn; c += 32) bias[c] = p.bias && c < own ? __ldg(p.bias + own0 + c) : 0.f;
            __syncwarp();
            const int half = done % T::kSums;
            if (!__all_sync(0xffffffffu, wait(&sums_done[half], done / T::kSums & 1))) break;
            tensor_fence_after();
            const uint32_t sums = memory + ((uint32_t)quarter << 21) + half * BN + c0;
            for (int c = 0; c < own; c += 32) {
                float v[32];
                load_sums32(sums + c, v);
                finish_sums<false, true>(p, v, 1.f, bias + c, nullptr, true);
                if (p.boxes) {
                    const bool starts = c % width == 0, ends = (c + 32) % width == 0 || c + 32 >= own;
                    if (starts) {
                        if (adds) {
                            if (c > 0) fetch_residual(c);
                            if (!__all_sync(0xffffffffu, wait(&residual_in[taker], residuals & 1))) break;
                            residuals++;
                        } else {
                            if (lane == 0) bulk_wait_read<0>();
                            __syncwarp();
                        }
                    }
                    unsigned char* row = box + lane * 128;
                    if (wide)
                        box_out<float>(row, lane, 0, v, adds);
                    else if (p.d_type == B200_TYPE_BF16)
                        box_out<bf16>(row, lane, starts ? 0 : 4, v, adds);
                    else
                        box_out<f16>(row, lane, starts ? 0 : 4, v, adds);
                    if (ends) {
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            store_box3(&d_map, smem_u32(box), (int)own0 + c / width * width, (int)rows0, 0);
                            bulk_commit();
                        }
                        __syncwarp();
                    }
                } else {  // through the box as fp32, a row of 32 elements at a time
                    box_out<float>(box + lane * 128, lane, 0, v, false);
                    __syncwarp();
                    if (c + lane < own) {
                        if (p.d_type == B200_TYPE_F32)
                            column_out<float>(p, box, lane, rows0, own0 + c + lane, adds);
                        else if (p.d_type == B200_TYPE_BF16)
                            column_out<bf16>(p, box, lane, rows0, own0 + c + lane, adds);
                        else
                            column_out<f16>(p, box, lane, rows0, own0 + c + lane, adds);
                    }
                    __syncwarp();
                }
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(PAIR ? of_rank(smem_u32(&sums_free[half]), 0) : smem_u32(&sums_free[half]));
        }
        if (lane == 0) bulk_wait_all();
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
