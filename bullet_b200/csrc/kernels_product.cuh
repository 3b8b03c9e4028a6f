// Products of matrices for the dense trunk, on the tensor pipe.
//
//   d[m][n] = act(scale * sum over k of a(m, k) b(k, n) + bias[n]) + residual[m][n]
//
// a and b lie in memory either along k (a row of consecutive k per m or n) or across (a row of consecutive m or n per k): a
// layer's forward is x along, W across; the gradient at its input dz along, W along; the gradient at its weights x across, dz
// across.  The tensor pipe takes both, so nothing is transposed.
//
// A CTA (or, PAIR, a pair of two SMs that share a tile of 256 rows and each fetch half of its columns) takes items, a tile of
// the result times a piece of k, one after another.  One thread has TMA fetch boxes of 128 bytes by rows, with the 128-byte
// swizzle, into a ring of stages; one issues the products of a stage as it arrives, with sums in tensor memory; kTakers warps take
// finished sums out, a thread a row, while the products of the next item go to the other half of tensor memory (tiles of 512 columns
// fill all of it, and their products wait), and hand them to TMA in boxes of 32 rows of 128 bytes, in which the residual lies already.
// With k cut (`parts`) the pieces' sums go to memory in fp32 and join_kernel adds them up in order.
//
// CODES: a is an 8-bit checkpoint with a scale per k.  Twelve more warps (kGroups of four) turn its codes into bf16 on the way from one place in
// shared memory to another: a power of two as scale makes that exact, so there is no product of other values than those
// that the checkpoint stands for, and no copy of it in 16 bits in memory.  (With other scales the values are rounded to bf16.)
#pragma once
#include "launch.cuh"
#include "tensor.cuh"
#include "values.cuh"

namespace b200 {

// The tensor pipe cuts sums off where it adds to them, so that long sums lose: 131072 products of checkpoints and gradients, the sums'
// error in 1 chain of 2048 stages 4e-5 of them, 228 stages 2.3e-6, 114 9e-7 (added up in fp32, 1.6e-7).  A sum is taken out after
// kChainMost stages and added, rounded, to what memory holds.
constexpr int kChainMost = 128;

struct ProductArgs {
    int64_t m, n, k;
    int tiles_m, tiles_n, k_blocks, blocks_per_item, parts_n;  // parts_n: pieces of k
    int chain;                                                 // stages that are added up in tensor memory (kChainMost)
    uint32_t form_type;                                        // of product_form
    const float* a_scale;                                      // per m (products of 8 bits) or per k (CODES)
    const float* b_scale;                                      // per n (products of 8 bits)
    const float* bias;
    const void* residual;
    int64_t ldr;
    void* d;
    int64_t ldd;
    int d_type, act;
    int boxes;     // rows of d start and end on 16 bytes, those of the residual start on them: TMA takes them; else element by element
    float* parts;  // [parts_n][m][ldp], ldp = n up to a multiple of 8; null: none, there is one part of one chain
    int64_t ldp;
    int* gave_up;
    // The kernel before it on the stream is one of the same call whose result it does not read (the bias's sums joined, the other product
    // of a gradient): it starts while that one's last CTAs run, on the SMs that they leave over, and waits for it at the end instead.
    // Gradients, us: 5003 rows, 2048 -> 1024 73.6 without, 69.7 beside the other product; 16384 rows, 512 -> 256 47.6 and 43.0; 131072
    // rows, 2048 -> 512 605 and 602.  Beside the joined sums as well: 2000 rows, 512 -> 512 36.6 and 35.3, 5003 rows 70.0 and 69.6.
    int beside;
};

template <int BN, bool PAIR, bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
struct Tile {
    static constexpr int kColumns = BN, kRows = PAIR ? 256 : 128;
    static constexpr int kWide = BN == 512 ? 2 : 1;          // products of 256 columns side by side
    static constexpr int kOwnColumns = PAIR ? 128 : BN;      // of b, that this CTA fetches for each
    static constexpr int kBlock = BYTES ? 128 : 64;          // of k in a stage: 128 bytes
    static constexpr uint32_t kA = 128 * 128, kBOne = kOwnColumns * 128, kB = kWide * kBOne, kRaw = CODES ? 64 * 128 : 0, kStage = kA + kB;
    static constexpr int kTakers = BN == 64 || CODES ? 4 : 8;  // warps that take sums out
    static constexpr int kOwn = BN * 4 / kTakers;              // columns of each of them
    static constexpr bool kColumnValues = B_ACROSS && !A_ACROSS;  // a bias, and scales of 8-bit weights
    static constexpr int kGroups = CODES ? 3 : 0;              // of four warps that turn codes into bf16, a stage by turns
    static constexpr int kRaws = BN == 64 || BN == 512 ? kGroups : 2 * kGroups;  // codes on their way: a ring of their own
    static constexpr int kThreads = 64 + 32 * (kTakers + 4 * kGroups + (CODES ? 1 : 0));
    static constexpr int kBoxesEach = CODES ? 2 : 1;           // of the result on their way out (a chain's sums have to make room)
    static constexpr size_t kBoxes = kTakers * kBoxesEach * 4096;
    static constexpr size_t kValues = kColumnValues ? (size_t)kTakers * 2 * kOwn * 4 : 0;
    static constexpr size_t kRest = 1024 + kBoxes + kValues + kRaws * kRaw;
    static constexpr int kFit = (int)((232448 - 1024 - kRest) / kStage), kStages = kFit < 8 ? kFit : 8;  // (1 KB for barriers)
    static constexpr size_t kShared = kRest + (size_t)kStages * kStage;
    static constexpr int kSums = BN == 512 ? 1 : 2;            // items whose sums there is room for
    static constexpr uint32_t kMemory = kSums * BN;            // columns of tensor memory
    static_assert(!(BYTES && B_ACROSS) || kOwnColumns % 128 == 0, "boxes across are 128 bytes wide");
    static_assert(!CODES || (A_ACROSS && !BYTES), "");
    // A group has places of the ring of codes to itself, so that it is never more than one use of a place behind or ahead; and the
    // products that were before the last ones in the place of the stage it writes next have been waited for.
    static_assert(kGroups <= kStages && kStages >= 3, "");
};

// Four codes to bf16, times f.  A code's bits, moved to bf16's, are its value times 2^-120 (but NaN's, which would be 480).
__device__ __forceinline__ void codes_to_bf16(uint32_t w, __nv_bfloat162 f, uint32_t& low, uint32_t& high) {
    uint32_t t[2] = {__byte_perm(w, 0, 0x1404), __byte_perm(w, 0, 0x3424)};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t v = (t[h] & 0x80008000u) | (t[h] >> 4 & 0x07f007f0u);
        const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), f);
        t[h] = *reinterpret_cast<const uint32_t*>(&x);
    }
    low = t[0], high = t[1];
}
__device__ __forceinline__ uint32_t has_nan_code(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }  // & 0x80808080
// Four codes one by one into memory, rounded to bf16: for NaN, scales past 2^7 and scales that are no powers of two.
static __device__ __noinline__ void codes_to_bf16_slowly(uint32_t w, float scale, uint32_t* to) {
#pragma unroll 1
    for (int q = 0; q < 4; q++) reinterpret_cast<bf16*>(to)[q] = __float2bfloat16_rn(to_float(e4m3{(uint8_t)(w >> 8 * q)}) * scale);
}

// (one function: 32 times in line it would stand in the way of the usual scales' code)
static __device__ __noinline__ float scaled_slowly(float v, float a, float b) { return scaled(v, a, b); }
// 32 sums of a row as whole sums end: scales, bias (of these columns, in shared memory), activation.  `usual`: all products of two
// scales that the warp meets are normal numbers.
template <bool BYTES, bool VALUES>
__device__ __forceinline__ void finish_sums(const ProductArgs& p, float (&v)[32], float a_scale, const float* bias, const float* b_scale, bool usual) {
    if constexpr (BYTES) {
        if (__builtin_expect(usual, 1)) {
#pragma unroll
            for (int g = 0; g < 8; g++) {
                const float4 b = reinterpret_cast<const float4*>(b_scale)[g];
                v[4 * g] *= a_scale * b.x, v[4 * g + 1] *= a_scale * b.y, v[4 * g + 2] *= a_scale * b.z, v[4 * g + 3] *= a_scale * b.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 32; k++) v[k] = scaled_slowly(v[k], a_scale, b_scale[k]);
        }
    }
    if constexpr (VALUES) {
#pragma unroll
        for (int g = 0; g < 8; g++) {
            const float4 b = reinterpret_cast<const float4*>(bias)[g];
            v[4 * g] += b.x, v[4 * g + 1] += b.y, v[4 * g + 2] += b.z, v[4 * g + 3] += b.w;
        }
        activate_all(v, p.act);
    }
}
// Half of a row of a box (16 bits: 32 columns of 64; fp32: 32 columns, the whole), the residual there added, in place.  Rows of 128 bytes
// in the 128-byte swizzle; `row`: its start, r its number.
template <class T>
__device__ __forceinline__ void box_out(unsigned char* row, int r, int first_piece, const float (&v)[32], bool residual) {
    constexpr int kPieces = sizeof(T) == 4 ? 8 : 4;
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        uint4* at = reinterpret_cast<uint4*>(row + (((first_piece + k) ^ (r & 7)) << 4));
        uint32_t w[4];
        if constexpr (sizeof(T) == 4) {
            float x[4] = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
            if (residual) {
                const float4 o = *reinterpret_cast<const float4*>(at);
                x[0] += o.x, x[1] += o.y, x[2] += o.z, x[3] += o.w;
            }
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = __float_as_uint(x[q]);
        } else {
            float x[8];
#pragma unroll
            for (int q = 0; q < 8; q++) x[q] = v[8 * k + q];
            if (residual) {
                const uint4 o = *at;
                const uint32_t u[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float low, high;
                    unpack2<T>(u[q], low, high);
                    x[2 * q] += low, x[2 * q + 1] += high;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = pack2<T>(x[2 * q], x[2 * q + 1]);
        }
        *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A column of a box of fp32, the residual added, element by element; sixteen of the residual are on their way at a time.
template <class T>
static __device__ __forceinline__ void column_out(const ProductArgs& p, const unsigned char* box, int lane, int64_t rows0, int64_t column, bool adds) {
    const T* residual = static_cast<const T*>(p.residual) + column;
    T* d = static_cast<T*>(p.d) + column;
    const int64_t last = p.m - 1;
    for (int r0 = 0; r0 < 32 && rows0 + r0 <= last; r0 += 16) {
        T added[16];
        if (adds)
#pragma unroll
            for (int r = 0; r < 16; r++) added[r] = residual[min(rows0 + r0 + r, last) * p.ldr];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const float x = *reinterpret_cast<const float*>(box + (r0 + r) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            if (rows0 + r0 + r <= last) d[(rows0 + r0 + r) * p.ldd] = from_float<T>(adds ? x + to_float(added[r]) : x);
        }
    }
}

template <int BN, bool PAIR, bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
static __global__ void __launch_bounds__((Tile<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>::kThreads), 1)
    product_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const __grid_constant__ CUtensorMap d_map,
                   const __grid_constant__ CUtensorMap r_map, const ProductArgs p) {
    using T = Tile<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>;
    constexpr int kStages = T::kStages, kCtas = PAIR ? 2 : 1;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t full[kStages], empty[kStages], ready[kStages], sums_done[2], sums_free[2], codes_in[T::kRaws + 1], codes_out[T::kRaws + 1], residual_in[T::kTakers];
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
            mbar_init(&ready[s], 4 * kCtas);
        }
        for (int s = 0; s < T::kRaws; s++) {
            mbar_init(&codes_in[s], 1);
            mbar_init(&codes_out[s], 4);
        }
        for (int k = 0; k < T::kTakers; k++) mbar_init(&residual_in[k], 1);
        for (int k = 0; k < 2; k++) {
            mbar_init(&sums_done[k], 1);
            mbar_init(&sums_free[k], T::kTakers * kCtas);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (threadIdx.x == 64 && p.beside) step_takes_over();  // (beside the preparations; the barrier below is behind it)
    if (threadIdx.x == 32) {
        know_map(&a_map);
        know_map(&b_map);
        if (p.boxes) know_map(&d_map);
    }
    __syncwarp();
    if (warp == 1) tensor_memory_take<PAIR>(&memory_at, T::kMemory);
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tensor_fence_after();
    const uint32_t memory = memory_at;
    // (behind the own memory and barriers: what a kernel of the same call left is read from here on; that before the one that it stands
    // beside, dz, has completed: dense_dz_kernel -> [joined sums of the bias ->] dx -> dw, and of these the first behind dense_dz_kernel
    // waits for it before it lets the next one in)
    if (!p.beside) step_waits();
    if (threadIdx.x == 32) step_hands_on();

    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, items = tiles * p.parts_n;
    const int64_t first = blockIdx.x / kCtas, step = gridDim.x / kCtas;
    auto item_of = [&](int64_t item, int64_t& m0, int64_t& n0, int& k0, int& k1, int& part) {
        part = (int)(item / tiles);
        const int64_t tile = item % tiles;
        m0 = tile / p.tiles_n * T::kRows;
        n0 = tile % p.tiles_n * BN;
        k0 = part * p.blocks_per_item;
        k1 = min(p.k_blocks, k0 + p.blocks_per_item);
    };
    int64_t m0, n0;
    int k0, k1, part;

    if (warp == 0) {
        if (lane == 0) {  // fetches
            int s = 0;
            uint32_t phase = 1;  // (a new barrier's phase before is over)
            for (int64_t item = first; item < items && !dead; item += step) {
                item_of(item, m0, n0, k0, k1, part);
                m0 += 128 * rank;
                n0 += PAIR ? 128 * rank : 0;
                for (int kb = k0; kb < k1; kb++) {
                    if (!wait(&empty[s], phase)) break;
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA;
                    const uint32_t bar = PAIR ? of_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
                    const int k = kb * T::kBlock;
                    if (rank == 0) mbar_expect_tx(&full[s], kCtas * (CODES ? T::kB : T::kA + T::kB));
                    if constexpr (CODES) {  // (others fetch and write a)
                    } else if constexpr (A_ACROSS) {
#pragma unroll
                        for (int c = 0; c < 128 / T::kBlock; c++) load_box<PAIR>(a_at + c * T::kBlock * 128, &a_map, (int)m0 + c * T::kBlock, k, bar);
                    } else {
                        load_box<PAIR>(a_at, &a_map, k, (int)m0, bar);
                    }
#pragma unroll
                    for (int h = 0; h < T::kWide; h++) {
                        if constexpr (B_ACROSS) {
#pragma unroll
                            for (int c = 0; c < T::kOwnColumns / T::kBlock; c++)
                                load_box<PAIR>(b_at + h * T::kBOne + c * T::kBlock * 128, &b_map, (int)n0 + 256 * h + c * T::kBlock, k, bar);
                        } else {
                            load_box<PAIR>(b_at + h * T::kBOne, &b_map, k, (int)n0 + 256 * h, bar);
                        }
                    }
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {  // multiplies
            constexpr uint32_t column = T::kBlock * 128;                                    // bytes from 128 bytes across to the next
            constexpr uint32_t a_step = A_ACROSS ? T::kBlock * 32 : 32, b_step = B_ACROSS ? T::kBlock * 32 : 32;  // a quarter of a stage's k
            const uint32_t form = product_form(p.form_type, A_ACROSS, B_ACROSS, T::kRows, BN / T::kWide);
            int s = 0, done = 0;
            uint32_t phase = 0;
            for (int64_t item = first; item < items && !dead; item += step) {
                item_of(item, m0, n0, k0, k1, part);
                bool fine = true;
                for (int kc = k0; kc < k1 && fine; kc += p.chain, done++) {
                    const int half = done % T::kSums;
                    const uint32_t sums = memory + half * BN;
                    fine = wait(&sums_free[half], (done / T::kSums & 1) ^ 1);
                    if (!fine) break;
                    tensor_fence_after();
                    for (int kb = kc; kb < min(kc + p.chain, k1); kb++) {
                        fine = wait(&full[s], phase) && (!CODES || wait(&ready[s], phase));
                        if (!fine) break;
                        tensor_fence_after();
                        const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA;
#pragma unroll
                        for (int q = 0; q < 4; q++)
#pragma unroll
                            for (int h = 0; h < T::kWide; h++)
                                multiply<PAIR, BYTES>(sums + 256 * h, tile_descriptor(a_at + q * a_step, A_ACROSS ? column : 16),
                                                      tile_descriptor(b_at + h * T::kBOne + q * b_step, B_ACROSS ? column : 16), form, kb > kc || q > 0);
                        when_multiplied<PAIR>(&empty[s]);
                        if (++s == kStages) s = 0, phase ^= 1;
                    }
                    when_multiplied<PAIR>(&sums_done[half]);
                }
            }
        }
    } else if (warp < 2 + T::kTakers) {  // takes sums out, kOwn columns of 32 rows
        const int quarter = warp & 3, taker = warp - 2, c0 = taker / 4 * T::kOwn;
        unsigned char* boxes = base + kStages * T::kStage + T::kRaws * T::kRaw + taker * T::kBoxesEach * 4096;
        unsigned char* box = boxes;
        float* bias = reinterpret_cast<float*>(base + kStages * T::kStage + T::kRaws * T::kRaw + T::kBoxes) + taker * 2 * T::kOwn;
        float* b_scale = bias + T::kOwn;
        const bool wide = p.boxes && (p.d_type == B200_TYPE_F32 || p.parts), adds = p.residual && !p.parts;
        const int width = wide ? 32 : 64;  // columns of a box
        uint32_t residuals = 0;
        int done = 0;
        bool fine = true;
        for (int64_t item = first; item < items && fine; item += step) {
            item_of(item, m0, n0, k0, k1, part);
            const int64_t rows0 = m0 + 128 * rank + 32 * quarter, m = rows0 + lane, own0 = n0 + c0;
            const int own = rows0 < p.m ? (int)min((int64_t)T::kOwn, p.n - own0) : 0;  // columns there are, 0 or less: nothing here
            const bool here = m < p.m;
            const float a_scale = BYTES && here ? __ldg(p.a_scale + m) : 1.f;
            auto fetch_residual = [&](int c) {
                if (lane == 0) {
                    bulk_wait_read<0>();
                    mbar_expect_tx(&residual_in[taker], 4096);
                    load_box3(smem_u32(box), &r_map, (int)own0 + c, (int)rows0, 0, smem_u32(&residual_in[taker]));
                }
            };
            if (adds && p.boxes && own > 0) fetch_residual(0);
            bool usual = true;
            if constexpr (T::kColumnValues) {
                __syncwarp();
                uint32_t least = 0x7f7fffffu, most = 0;  // of the scales, by their bits
                for (int c = lane; c < T::kOwn; c += 32) {
                    bias[c] = p.bias && c < own ? __ldg(p.bias + own0 + c) : 0.f;
                    if constexpr (BYTES) {
                        const float b = c < own ? __ldg(p.b_scale + own0 + c) : 0.f;
                        b_scale[c] = b;
                        const uint32_t size = __float_as_uint(b) & 0x7fffffffu;
                        if (c < own) least = min(least, size), most = max(most, size);
                    }
                }
                if constexpr (BYTES) {
                    least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
                    usual = __all_sync(0xffffffffu, normal(a_scale * __uint_as_float(least)) && normal(a_scale * __uint_as_float(most)));
                }
                __syncwarp();
            }
            for (int kc = k0; kc < k1; kc += p.chain, done++) {
                const int half = done % T::kSums;
                fine = __all_sync(0xffffffffu, wait(&sums_done[half], done / T::kSums & 1));
                if (!fine) break;
                if (kc > k0 && lane == 0) bulk_wait_all();  // what this part's chains before have left is in memory
                tensor_fence_after();
                const uint32_t sums = memory + ((uint32_t)quarter << 21) + half * BN + c0;
                for (int c = 0; c < own; c += 32) {
                    float v[32];
                    load_sums32(sums + c, v);
                    if (!p.parts) finish_sums<BYTES, T::kColumnValues>(p, v, a_scale, bias + c, b_scale + c, usual);
                    if (p.boxes) {
                        const bool starts = c % width == 0, ends = (c + 32) % width == 0 || c + 32 >= own;
                        if (starts) {
                            if (adds) {
                                if (c > 0) fetch_residual(c);
                                if (!__all_sync(0xffffffffu, wait(&residual_in[taker], residuals & 1))) break;
                                residuals++;
                            } else {
                                if constexpr (T::kBoxesEach == 2) box = box == boxes ? boxes + 4096 : boxes;
                                if (lane == 0) bulk_wait_read<T::kBoxesEach - 1>();
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
                                if (kc > k0)
                                    add_box3(&d_map, smem_u32(box), (int)own0 + c / width * width, (int)rows0, part);
                                else
                                    store_box3(&d_map, smem_u32(box), (int)own0 + c / width * width, (int)rows0, part);
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
        }
        if (lane == 0) bulk_wait_all();
    } else if (CODES && warp == T::kThreads / 32 - 1) {
        if (lane == 0) {  // fetches codes
            int s = 0;
            uint32_t phase = 1;
            for (int64_t item = first; item < items && !dead; item += step) {
                item_of(item, m0, n0, k0, k1, part);
                for (int kb = k0; kb < k1; kb++) {
                    if (!wait(&codes_out[s], phase)) break;
                    mbar_expect_tx(&codes_in[s], T::kRaw);
                    load_box<false>(smem_u32(base + kStages * T::kStage + s * T::kRaw), &a_map, (int)(m0 + 128 * rank), kb * T::kBlock, smem_u32(&codes_in[s]));
                    if (++s == T::kRaws) s = 0, phase ^= 1;
                }
            }
        }
    } else if constexpr (CODES) {  // 8 threads a row of 128 codes, 16 each
        const int t = (threadIdx.x - 64 - 32 * T::kTakers) & 127, row = t >> 3, j = t & 7, group = (warp - 2 - T::kTakers) >> 2;
        int s = 0, in = 0, turn = 0;  // whose stage it is
        uint32_t phase = 1, in_phase = 0;
        auto next = [&]() {
            if (++s == kStages) s = 0, phase ^= 1;
            if (++in == T::kRaws) in = 0, in_phase ^= 1;
        };
        for (int64_t item = first; item < items && !dead; item += step) {
            item_of(item, m0, n0, k0, k1, part);
            uint32_t scale[4];
            auto fetch = [&](int kb) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int64_t k = (int64_t)kb * 64 + row + 16 * i;
                    scale[i] = kb < k1 && k < p.k ? __float_as_uint(__ldg(p.a_scale + k)) : 127u << 23;
                }
            };
            fetch(k0 + (group + T::kGroups - turn) % T::kGroups);
            for (int kb = k0; kb < k1; kb++) {
                const bool mine = turn == group;
                if (++turn == T::kGroups) turn = 0;
                if (!mine) {
                    next();
                    continue;
                }
                if (!__all_sync(0xffffffffu, wait(&codes_in[in], in_phase))) break;
                const unsigned char* raw = base + kStages * T::kStage + in * T::kRaw + row * 128 + 16 * j;
                unsigned char* to = base + s * T::kStage + (j >> 2) * 8192 + row * 128;
                // (the upper half of the threads of a row write their second piece first: eight threads meet all banks)
                const int at0 = ((2 * (j & 3) + (j >> 2)) ^ (row & 7)) << 4, at1 = at0 ^ 16;
                uint4 code[4];
#pragma unroll
                for (int i = 0; i < 4; i++) code[i] = *reinterpret_cast<const uint4*>(raw + i * 2048);
                uint32_t nan = 0, v[4][8];
                bool slow = false;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t e = scale[i] >> 23;
                    slow |= scale[i] - (1u << 23) > 133u << 23 || (scale[i] & 0x7fffffu);  // (2^-126 to 2^7 are not)
                    const __nv_bfloat162 f = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)((min(e, 134u) + 120u) << 7)));
                    const uint4 c = j >> 2 ? make_uint4(code[i].z, code[i].w, code[i].x, code[i].y) : code[i];
                    nan |= has_nan_code(c.x) | has_nan_code(c.y) | has_nan_code(c.z) | has_nan_code(c.w);
                    codes_to_bf16(c.x, f, v[i][0], v[i][1]);
                    codes_to_bf16(c.y, f, v[i][2], v[i][3]);
                    codes_to_bf16(c.z, f, v[i][4], v[i][5]);
                    codes_to_bf16(c.w, f, v[i][6], v[i][7]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&codes_out[in]);
                if (!__all_sync(0xffffffffu, wait(&empty[s], phase))) break;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    *reinterpret_cast<uint4*>(to + i * 2048 + at0) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
                    *reinterpret_cast<uint4*>(to + i * 2048 + at1) = make_uint4(v[i][4], v[i][5], v[i][6], v[i][7]);
                }
                if (slow || nan & 0x80808080u) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            codes_to_bf16_slowly(w[q], __uint_as_float(scale[i]), reinterpret_cast<uint32_t*>(to + i * 2048 + ((j >> 2) ^ (q >> 1) ? at1 : at0) + (q & 1) * 8));
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive_at(PAIR ? of_rank(smem_u32(&ready[s]), 0) : smem_u32(&ready[s]));
                fetch(kb + T::kGroups);  // (behind the fence, which would wait for it)
                next();
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
        tensor_memory_give<PAIR>(memory, T::kMemory);
    }
    if (p.beside) step_waits();  // who waits for this kernel waits for both
}

// Pieces from `s` on, N of them on their way at a time, while there are as many.
template <int N>
__device__ __forceinline__ void add_pieces(const ProductArgs& p, const float* at, int& s, float (&v)[4]) {
    for (; s + N <= p.parts_n; s += N) {
        float4 f[N];
#pragma unroll
        for (int r = 0; r < N; r++) f[r] = __ldcs(reinterpret_cast<const float4*>(at + (s + r) * p.m * p.ldp));
#pragma unroll
        for (int r = 0; r < N; r++) v[0] += f[r].x, v[1] += f[r].y, v[2] += f[r].z, v[3] += f[r].w;
    }
}
// The pieces of k added up in order, and what finish_sums does to whole sums.  A thread takes four columns.  (What is on its way is said
// by add_pieces: a loop left to the compiler lost it to a little more code behind it, layer 9 x 8192 -> 64 12.6 -> 16.6 us, gradient of 16384
// rows, 512 -> 256 42.4 -> 44.3.)
template <bool BYTES>
static __global__ void __launch_bounds__(256) join_kernel(const ProductArgs p) {
    step_begin(nullptr);
    const int64_t per_row = p.ldp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.m * per_row) return;
    const int64_t m = i / per_row, n = i % per_row * 4;
    float v[4] = {};
    const float* at = p.parts + m * p.ldp + n;
    int s = 0;
    add_pieces<8>(p, at, s, v);
    add_pieces<4>(p, at, s, v);
    add_pieces<2>(p, at, s, v);
    add_pieces<1>(p, at, s, v);
    const float a_scale = BYTES ? p.a_scale[m] : 1.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (n + k >= p.n) return;
        float x = v[k];
        if constexpr (BYTES) x = scaled(x, a_scale, p.b_scale[n + k]);
        if (p.bias) x += p.bias[n + k];
        x = activate(x, p.act);
        if (p.residual) x += load_value(p.residual, m * p.ldr + n + k, p.d_type);
        store_value(p.d, m * p.ldd + n + k, p.d_type, x);
    }
}

// A matrix whose rows do not start on 16 bytes, copied to one whose rows do, side by side.  A thread puts 16 bytes together out of the
// five words of four that they lie in, of which it loads those that hold any byte of the row.
constexpr int kAlignPieces = 4;  // of a thread, in flight
static __global__ void __launch_bounds__(256) align_rows_kernel(const uint8_t* from, int64_t apart, uint4* to, int64_t rows, int64_t bytes) {
    const int64_t per_row = (bytes + 15) / 16, all = rows * per_row;
    uint32_t w[kAlignPieces][5];
    int shift[kAlignPieces];
#pragma unroll
    for (int q = 0; q < kAlignPieces; q++) {
        const int64_t i = (int64_t)blockIdx.x * 256 * kAlignPieces + q * 256 + threadIdx.x;
        if (i >= all) continue;
        const uint8_t* row = from + i / per_row * apart;
        const uint8_t* at = row + i % per_row * 16;
        const uint32_t* words = reinterpret_cast<const uint32_t*>((uintptr_t)at & ~(uintptr_t)3);
        shift[q] = 8 * (int)((uintptr_t)at & 3);
#pragma unroll
        for (int k = 0; k < 5; k++) w[q][k] = reinterpret_cast<const uint8_t*>(words + k) < row + bytes ? words[k] : 0u;
    }
#pragma unroll
    for (int q = 0; q < kAlignPieces; q++) {
        const int64_t i = (int64_t)blockIdx.x * 256 * kAlignPieces + q * 256 + threadIdx.x;
        if (i < all)
            to[i] = make_uint4(__funnelshift_r(w[q][0], w[q][1], shift[q]), __funnelshift_r(w[q][1], w[q][2], shift[q]), __funnelshift_r(w[q][2], w[q][3], shift[q]),
                               __funnelshift_r(w[q][3], w[q][4], shift[q]));
    }
}

// dz = act'(y) * dy, rounded to dy's type (dz: rows of ldz, or null), and the sums of the unrounded values over pieces of the
// rows: parts[piece][out] (or null).  HBM bound.  The threads of a CTA are `across` side by side, V columns each.
template <class TD, class TY, int V>
static __global__ void __launch_bounds__(256) dense_dz_kernel(b200_dense_grad_op a, TD* dz, int64_t ldz, float* parts, int across) {
    constexpr int kAhead = 8;  // rows (131072 x 2048 from 8-bit outputs: 4 260 us, 8 228)
    __shared__ float added[256 * V];
    step_begin(nullptr);
    const int lane = (int)threadIdx.x % across, column = (blockIdx.x * across + lane) * V, step = 256 / across;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    const TD* dy = static_cast<const TD*>(a.dy) + column;
    const TY* y = static_cast<const TY*>(a.y) + column;
    float sum[V] = {};
    if (column < a.out) {
        for (int64_t row = first + (int)threadIdx.x / across; row < last; row += step * kAhead) {
            TD g[kAhead][V];
            TY o[kAhead][V];
            float scale[kAhead];
#pragma unroll
            for (int r = 0; r < kAhead; r++) {
                const int64_t at = min(row + r * step, last - 1);
                if constexpr (V == 8) {
                    *reinterpret_cast<uint4*>(g[r]) = __ldcs(reinterpret_cast<const uint4*>(dy + at * a.lddy));
                    if (a.act != B200_ACT_NONE) {
                        if constexpr (sizeof(TY) == 1)
                            *reinterpret_cast<uint2*>(o[r]) = __ldcs(reinterpret_cast<const uint2*>(y + at * a.ldy));
                        else
                            *reinterpret_cast<uint4*>(o[r]) = __ldcs(reinterpret_cast<const uint4*>(y + at * a.ldy));
                    }
                } else {
                    g[r][0] = dy[at * a.lddy];
                    if (a.act != B200_ACT_NONE) o[r][0] = y[at * a.ldy];
                }
                scale[r] = sizeof(TY) == 1 && a.act != B200_ACT_NONE ? __ldg(a.y_scale + at) : 1.f;
            }
#pragma unroll
            for (int r = 0; r < kAhead; r++) {
                if (row + r * step >= last) break;
                TD out[V];
#pragma unroll
                for (int k = 0; k < V; k++) {
                    float v = to_float(g[r][k]);
                    if (a.act != B200_ACT_NONE) v = gradient_from_output(v, to_float(o[r][k]) * scale[r], a.act);
                    sum[k] += v;
                    out[k] = from_float<TD>(v);
                }
                if (dz) {
                    if constexpr (V == 8)
                        *reinterpret_cast<uint4*>(dz + (row + r * step) * ldz + column) = *reinterpret_cast<const uint4*>(out);
                    else
                        dz[(row + r * step) * ldz + column] = out[0];
                }
            }
        }
    }
    if (!parts) return;
#pragma unroll
    for (int k = 0; k < V; k++) added[k * 256 + threadIdx.x] = sum[k];
    __syncthreads();
    for (int c = threadIdx.x; c < across * V; c += 256) {
        const int n = blockIdx.x * across * V + c;
        if (n >= a.out) break;
        float v = 0.f;
        for (int r = 0; r < step; r++) v += added[c % V * 256 + r * across + c / V];
        parts[(int64_t)blockIdx.y * a.out + n] = v;
    }
}

}  // namespace b200
