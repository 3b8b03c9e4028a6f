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
// swizzle, into a ring of stages; one issues the products of a stage as it arrives, with sums in tensor memory; four warps take
// finished sums out, a thread a row, while the products of the next item go to the other half of tensor memory.  Their stores are whole
// 32-byte sectors.  With k cut (`parts`) the pieces' sums go to memory in fp32 and join_kernel adds them up in order.
//
// CODES: a is an 8-bit checkpoint with a scale per k.  Four more warps turn its codes into bf16 on the way from one place in
// shared memory to another: a power of two as scale makes that exact, so there is no product of other values than those
// that the checkpoint stands for, and no copy of it in 16 bits in memory.
#pragma once
#include "tensor.cuh"
#include "values.cuh"

namespace b200 {

struct ProductArgs {
    int64_t m, n, k;
    int tiles_m, tiles_n, k_blocks, blocks_per_item, parts_n;  // parts_n: pieces of k
    uint32_t form_type;                                        // of product_form
    const float* a_scale;                                      // per m (products of 8 bits) or per k (CODES)
    const float* b_scale;                                      // per n (products of 8 bits)
    const float* bias;
    const void* residual;
    int64_t ldr;
    void* d;
    int64_t ldd;
    int d_type, act;
    int wide;      // rows of d and of the residual start on 16 bytes; 2: of d on 32
    float* parts;  // [parts_n][m][ldp], ldp = n up to a multiple of 8; null: none
    int64_t ldp;
    int* gave_up;
};

template <int BN, bool PAIR, bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
struct Tile {
    static constexpr int kColumns = BN, kRows = PAIR ? 256 : 128;
    static constexpr int kOwnColumns = PAIR ? BN / 2 : BN;   // of b, that this CTA fetches
    static constexpr int kBlock = BYTES ? 128 : 64;          // of k in a stage: 128 bytes
    static constexpr uint32_t kA = 128 * 128, kB = kOwnColumns * 128, kRaw = CODES ? 64 * 128 : 0, kStage = kA + kB + kRaw;
    static constexpr int kStages = PAIR || BN == 128 ? 196608 / kStage : 98304 / kStage;  // (two CTAs of the narrowest tile fit on an SM)
    static constexpr int kThreads = CODES ? 320 : 192;
    static constexpr size_t kShared = 1024 + (size_t)kStages * kStage;
    static constexpr uint32_t kMemory = 2 * BN;  // columns of tensor memory
    static_assert(!(BYTES && B_ACROSS) || kOwnColumns % 128 == 0, "boxes across are 128 bytes wide");
    static_assert(!CODES || (A_ACROSS && !BYTES), "");
};

// Four codes to bf16, times f (powers of two; `more`: and g).  A code's bits, moved to bf16's, are its value times 2^-120.
__device__ __forceinline__ void codes_to_bf16(uint32_t w, __nv_bfloat162 f, bool more, __nv_bfloat162 g, uint32_t& low, uint32_t& high) {
    uint32_t t[2] = {__byte_perm(w, 0, 0x1404), __byte_perm(w, 0, 0x3424)};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t v = (t[h] & 0x80008000u) | ((t[h] & 0x7f007f00u) >> 4);
        __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), f);
        if (more) x = __hmul2(x, g);
        t[h] = *reinterpret_cast<const uint32_t*>(&x);
    }
    low = t[0], high = t[1];
}
__device__ __forceinline__ uint32_t has_nan_code(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }  // & 0x80808080

// What becomes of eight sums of a row, all inside the result: d and the residual on 16 bytes.
template <class T>
__device__ __forceinline__ void finish_eight(const float (&v)[32], int g, T* d, const T* residual, bool two_sectors) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = v[8 * g + k];
    if (residual) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float4 r = __ldg(reinterpret_cast<const float4*>(residual) + k);
                x[4 * k] += r.x, x[4 * k + 1] += r.y, x[4 * k + 2] += r.z, x[4 * k + 3] += r.w;
            }
        } else {
            const uint4 r = __ldg(reinterpret_cast<const uint4*>(residual));
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float low, high;
                unpack2<T>(w[k], low, high);
                x[2 * k] += low, x[2 * k + 1] += high;
            }
        }
    }
    if constexpr (sizeof(T) == 4) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; k++) w[k] = __float_as_uint(x[k]);
        if (two_sectors) {
            store_32_bytes(d, w);
        } else {
            reinterpret_cast<uint4*>(d)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(d)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
        *reinterpret_cast<uint4*>(d) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}
template <class T>
__device__ __forceinline__ void finish_typed(const ProductArgs& p, const float (&v)[32], int count, T* d, const T* residual) {
    if (p.wide) {
        if constexpr (sizeof(T) == 2) {
            if (count == 32 && p.wide == 2) {  // whole sectors
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t w[8], r[8] = {};
                    if (residual) {
                        const uint4 r0 = __ldg(reinterpret_cast<const uint4*>(residual + 16 * h)), r1 = __ldg(reinterpret_cast<const uint4*>(residual + 16 * h) + 1);
                        r[0] = r0.x, r[1] = r0.y, r[2] = r0.z, r[3] = r0.w, r[4] = r1.x, r[5] = r1.y, r[6] = r1.z, r[7] = r1.w;
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        float low, high;
                        unpack2<T>(r[k], low, high);
                        w[k] = residual ? pack2<T>(v[16 * h + 2 * k] + low, v[16 * h + 2 * k + 1] + high) : pack2<T>(v[16 * h + 2 * k], v[16 * h + 2 * k + 1]);
                    }
                    store_32_bytes(d + 16 * h, w);
                }
                return;
            }
        }
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (8 * g + 8 <= count) finish_eight<T>(v, g, d + 8 * g, residual ? residual + 8 * g : nullptr, p.wide == 2);
    }
    const int from = p.wide ? count & ~7 : 0;
#pragma unroll
    for (int k = 0; k < 32; k++)
        if (k >= from && k < count) d[k] = from_float<T>(residual ? v[k] + to_float(residual[k]) : v[k]);
}
// What becomes of 32 sums of a row, from column n on.
__device__ __forceinline__ void finish_sums(const ProductArgs& p, int part, int64_t m, int64_t n, float (&v)[32], float a_scale) {
    const int count = (int)min((int64_t)32, p.n - n);
    if (p.parts) {
        float* at = p.parts + (part * p.m + m) * p.ldp + n;
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (8 * g < count) {  // (rows have room for eights)
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; k++) w[k] = __float_as_uint(v[8 * g + k]);
                store_32_bytes(at + 8 * g, w);
            }
        return;
    }
    if (p.b_scale)
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] *= a_scale * (k < count ? __ldg(p.b_scale + n + k) : 0.f);
    if (p.bias)
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] += k < count ? __ldg(p.bias + n + k) : 0.f;
    if (p.act != B200_ACT_NONE)
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = activate(v[k], p.act);
    const int64_t d_at = m * p.ldd + n, r_at = m * p.ldr + n;
    if (p.d_type == B200_TYPE_F32)
        finish_typed(p, v, count, static_cast<float*>(p.d) + d_at, p.residual ? static_cast<const float*>(p.residual) + r_at : nullptr);
    else if (p.d_type == B200_TYPE_BF16)
        finish_typed(p, v, count, static_cast<bf16*>(p.d) + d_at, p.residual ? static_cast<const bf16*>(p.residual) + r_at : nullptr);
    else
        finish_typed(p, v, count, static_cast<f16*>(p.d) + d_at, p.residual ? static_cast<const f16*>(p.residual) + r_at : nullptr);
}

template <int BN, bool PAIR, bool BYTES, bool A_ACROSS, bool B_ACROSS, bool CODES>
static __global__ void __launch_bounds__((Tile<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>::kThreads), 1)
    product_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const ProductArgs p) {
    using T = Tile<BN, PAIR, BYTES, A_ACROSS, B_ACROSS, CODES>;
    constexpr int kStages = T::kStages, kCtas = PAIR ? 2 : 1;
    extern __shared__ unsigned char raw_smem[];
    __shared__ uint64_t full[kStages], empty[kStages], codes_in[kStages], ready[kStages], sums_done[2], sums_free[2];
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
            mbar_init(&codes_in[s], 1);
            mbar_init(&ready[s], 4 * kCtas);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&sums_done[k], 1);
            mbar_init(&sums_free[k], 4 * kCtas);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 1) tensor_memory_take<PAIR>(&memory_at, T::kMemory);
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tensor_fence_after();
    const uint32_t memory = memory_at;

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
                n0 += T::kOwnColumns * rank;
                for (int kb = k0; kb < k1; kb++) {
                    if (!wait(&empty[s], phase)) break;
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA, raw_at = b_at + T::kB;
                    const uint32_t bar = PAIR ? of_rank(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
                    const int k = kb * T::kBlock;
                    if (rank == 0) mbar_expect_tx(&full[s], kCtas * (CODES ? T::kB : T::kA + T::kB));
                    if constexpr (CODES) {
                        mbar_expect_tx(&codes_in[s], T::kRaw);
                        load_box<false>(raw_at, &a_map, (int)m0, k, smem_u32(&codes_in[s]));
                    } else if constexpr (A_ACROSS) {
#pragma unroll
                        for (int c = 0; c < 128 / T::kBlock; c++) load_box<PAIR>(a_at + c * T::kBlock * 128, &a_map, (int)m0 + c * T::kBlock, k, bar);
                    } else {
                        load_box<PAIR>(a_at, &a_map, k, (int)m0, bar);
                    }
                    if constexpr (B_ACROSS) {
#pragma unroll
                        for (int c = 0; c < T::kOwnColumns / T::kBlock; c++) load_box<PAIR>(b_at + c * T::kBlock * 128, &b_map, (int)n0 + c * T::kBlock, k, bar);
                    } else {
                        load_box<PAIR>(b_at, &b_map, k, (int)n0, bar);
                    }
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {  // multiplies
            constexpr uint32_t column = T::kBlock * 128;                                    // bytes from 128 bytes across to the next
            constexpr uint32_t a_step = A_ACROSS ? T::kBlock * 32 : 32, b_step = B_ACROSS ? T::kBlock * 32 : 32;  // a quarter of a stage's k
            const uint32_t form = product_form(p.form_type, A_ACROSS, B_ACROSS, T::kRows, BN);
            int s = 0, done = 0;
            uint32_t phase = 0;
            for (int64_t item = first; item < items && !dead; item += step, done++) {
                item_of(item, m0, n0, k0, k1, part);
                const int half = done & 1;
                const uint32_t sums = memory + half * BN;
                if (!wait(&sums_free[half], (done >> 1 & 1) ^ 1)) break;
                tensor_fence_after();
                bool fine = true;
                for (int kb = k0; kb < k1 && fine; kb++) {
                    fine = wait(&full[s], phase) && (!CODES || wait(&ready[s], phase));
                    if (!fine) break;
                    tensor_fence_after();
                    const uint32_t a_at = smem_u32(base + s * T::kStage), b_at = a_at + T::kA;
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        multiply<PAIR, BYTES>(sums, tile_descriptor(a_at + q * a_step, A_ACROSS ? column : 16), tile_descriptor(b_at + q * b_step, B_ACROSS ? column : 16), form,
                                              kb > k0 || q > 0);
                    when_multiplied<PAIR>(&empty[s]);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                when_multiplied<PAIR>(&sums_done[half]);
            }
        }
    } else if (warp < 6) {  // takes sums out
        const int quarter = warp & 3;
        int done = 0;
        for (int64_t item = first; item < items; item += step, done++) {
            item_of(item, m0, n0, k0, k1, part);
            const int half = done & 1;
            const int64_t m = m0 + 128 * rank + 32 * quarter + lane;
            const bool here = m < p.m;
            const float a_scale = BYTES && here && !p.parts ? __ldg(p.a_scale + m) : 1.f;
            const bool fine = __all_sync(0xffffffffu, wait(&sums_done[half], done >> 1 & 1));
            if (!fine) break;
            tensor_fence_after();
            for (int c = 0; c < BN / 32 && n0 + 32 * c < p.n; c++) {
                float v[32];
                load_sums32(memory + ((uint32_t)quarter << 21) + half * BN + 32 * c, v);
                if (here) finish_sums(p, part, m, n0 + 32 * c, v, a_scale);
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(PAIR ? of_rank(smem_u32(&sums_free[half]), 0) : smem_u32(&sums_free[half]));
        }
    } else if constexpr (CODES) {  // 8 threads a row of 128 codes, 16 each
        const int t = threadIdx.x - 192, row = t >> 3, j = t & 7;
        int s = 0;
        uint32_t phase = 0;
        for (int64_t item = first; item < items && !dead; item += step) {
            item_of(item, m0, n0, k0, k1, part);
            uint32_t scale[4];
            auto fetch = [&](int kb) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int64_t k = (int64_t)kb * 64 + row + 16 * i;
                    scale[i] = kb < k1 && k < p.k ? __float_as_uint(__ldg(p.a_scale + k)) >> 23 : 127u;
                }
            };
            fetch(k0);
            for (int kb = k0; kb < k1; kb++) {
                if (!__all_sync(0xffffffffu, wait(&codes_in[s], phase))) break;
                const unsigned char* raw = base + s * T::kStage + T::kA + T::kB;
                unsigned char* to = base + s * T::kStage + (j >> 2) * 8192;
                uint4 code[4];
#pragma unroll
                for (int i = 0; i < 4; i++) code[i] = *reinterpret_cast<const uint4*>(raw + (row + 16 * i) * 128 + 16 * j);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = (int)scale[i] - 127, most = min(e, 7);
                    const __nv_bfloat162 f = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)((most + 247) << 7)));
                    const __nv_bfloat162 g = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)((e - most + 127) << 7)));
                    const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
                    uint32_t v[8];
#pragma unroll
                    for (int q = 0; q < 4; q++) codes_to_bf16(w[q], f, e > 7, g, v[2 * q], v[2 * q + 1]);
                    if ((has_nan_code(w[0]) | has_nan_code(w[1]) | has_nan_code(w[2]) | has_nan_code(w[3])) & 0x80808080u)
#pragma unroll
                        for (int q = 0; q < 16; q++)
                            if ((w[q >> 2] >> 8 * (q & 3) & 0x7f) == 0x7f) v[q >> 1] |= 0x7fffu << 16 * (q & 1);
                    const int r = row + 16 * i;
                    // (the upper half of the threads of a row write their second piece first: eight threads meet all banks)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int piece = h ^ (j >> 2);
                        *reinterpret_cast<uint4*>(to + r * 128 + (((2 * (j & 3) + piece) ^ (r & 7)) << 4)) =
                            piece ? make_uint4(v[4], v[5], v[6], v[7]) : make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                fetch(kb + 1);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive_at(PAIR ? of_rank(smem_u32(&ready[s]), 0) : smem_u32(&ready[s]));
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
        tensor_memory_give<PAIR>(memory, T::kMemory);
    }
}

// The pieces of k added up in order, and what finish_sums does to whole sums.  A thread takes four columns.
static __global__ void __launch_bounds__(256) join_kernel(const ProductArgs p) {
    const int64_t per_row = p.ldp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.m * per_row) return;
    const int64_t m = i / per_row, n = i % per_row * 4;
    float v[4] = {};
    const float* at = p.parts + m * p.ldp + n;
#pragma unroll 4
    for (int s = 0; s < p.parts_n; s++) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(at + s * p.m * p.ldp));
        v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
    }
    const float a_scale = p.b_scale ? p.a_scale[m] : 1.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (n + k >= p.n) return;
        float x = v[k];
        if (p.b_scale) x *= a_scale * p.b_scale[n + k];
        if (p.bias) x += p.bias[n + k];
        x = activate(x, p.act);
        if (p.residual) x += load_value(p.residual, m * p.ldr + n + k, p.d_type);
        store_value(p.d, m * p.ldd + n + k, p.d_type, x);
    }
}

// A matrix whose rows do not start on 16 bytes, copied to one whose rows do.  E: bytes of an element.
template <class E>
static __global__ void __launch_bounds__(256) align_rows_kernel(const E* from, int64_t ld, E* to, int64_t ld_to, int64_t rows, int64_t cols) {
    const int64_t per = (cols + 255) / 256, i = blockIdx.x;
    const int64_t row0 = i / per * 8, c = i % per * 256 + threadIdx.x;
    if (c >= cols) return;
    E v[8];
#pragma unroll
    for (int r = 0; r < 8; r++) v[r] = from[min(row0 + r, rows - 1) * ld + c];
#pragma unroll
    for (int r = 0; r < 8; r++)
        if (row0 + r < rows) to[(row0 + r) * ld_to + c] = v[r];
}

// dz = act'(y) * dy, rounded to dy's type (dz: rows of ldz, or null), and the sums of the unrounded values over pieces of the
// rows: parts[piece][out] (or null).  HBM bound.  The threads of a CTA are `across` side by side, V columns each.
template <class TD, class TY, int V>
static __global__ void __launch_bounds__(256) dense_dz_kernel(b200_dense_grad_op a, TD* dz, int64_t ldz, float* parts, int across) {
    constexpr int kAhead = 4;
    __shared__ float added[256 * V];
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
