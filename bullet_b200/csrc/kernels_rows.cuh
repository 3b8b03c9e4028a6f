// Kernels over the rows of a matrix: root-mean-square norm and its gradient, 8-bit packing.
//
// With many rows all of them are bound by HBM but the norm to 8 bits, whose work per element shows beside it (16384 fp32 rows of 2048 37.6 us
// for 25.6 of traffic, 131072 bf16 rows with residual 306 for 287); with few rows latency counts.  A row is read once: W warps hold it in
// registers, NV vectors of eight elements a lane, from its first load to the last store, so that the norm's sum, the largest
// magnitude for the scale and the codes cost no second pass.  One warp takes up to 2048 columns by itself in packing, 1024 in a norm of
// 16 bits, 512 in one of fp32 and in the gradient (no barrier anywhere); wider rows, and narrower ones when there are too few rows for a
// warp each to fill the GPU, are shared by the warps of a CTA.  A vector's elements lie side by side where rows start on 16 bytes, else 32 apart, so that
// loads of single elements are coalesced.  Rows that do not fit in registers are taken by the *_any_ kernels, a CTA per row,
// in passes over L2.
#pragma once
#include <cuda_runtime.h>

#include <type_traits>

#include "launch.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kRowThreads = 256;
constexpr int kRowWarpsMost = 8;  // of a row

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Over the `warps` warps of a row; the same bits in every thread.  `shared`: one word per warp of the CTA, and not the words of the call
// before.  SEVERAL rows share a CTA, warps side by side; else a row of more than one warp has it to itself.  (Barriers by number: with
// a number out of a register a CTA counts as using all sixteen, and half as many CTAs fit on an SM.)
template <bool SEVERAL>
__device__ __forceinline__ void row_sync(int warps) {
    if constexpr (SEVERAL) {
        const int group = (int)(threadIdx.x >> 5) / warps;
        if (group == 0)
            asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
        else if (group == 1)
            asm volatile("bar.sync 2, %0;" ::"r"(32 * warps) : "memory");
        else if (group == 2)
            asm volatile("bar.sync 3, %0;" ::"r"(32 * warps) : "memory");
        else
            asm volatile("bar.sync 4, %0;" ::"r"(32 * warps) : "memory");
    } else {
        __syncthreads();
    }
}
template <bool SEVERAL = false>
__device__ __forceinline__ float row_sum(float v, int warps, float* shared) {
    v = warp_sum(v);
    if (warps == 1) return v;
    const int warp = threadIdx.x >> 5, first = SEVERAL ? warp / warps * warps : 0;
    if ((threadIdx.x & 31) == 0) shared[warp] = v;
    row_sync<SEVERAL>(warps);
    v = 0.f;
    for (int k = 0; k < warps; k++) v += shared[first + k];
    return v;
}
__device__ __forceinline__ uint32_t row_max(uint32_t v, int warps, uint32_t* shared) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int k = 0; k < warps; k++) v = max(v, shared[k]);
    return v;
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_magnitude(float v) { return finite(v) ? magnitude_bits(v) : 0u; }

// 32 bytes of a lane: neighbouring lanes' stand side by side, where two loads of 16 bytes would take twice the way through L1.  `stream`: not
// to be read again.
template <bool STREAM>
__device__ __forceinline__ void load_32_bytes(const void* at, uint32_t (&w)[8]) {
    if constexpr (STREAM)
        asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(at));
    else
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(at));
}
// Whether all of eight elements 32 apart are there: all but a row's last eights, which alone are looked at one by one.
__device__ __forceinline__ bool whole_eight(int first, int cols) { return first + 7 * 32 < cols; }
// Eight elements from `first` on (VEC) or from `first` on in steps of 32; those at or past `cols` are 0.
template <bool VEC, class T>
struct Eight {
    static constexpr int kWords = sizeof(T) / 2;  // of 16 bytes
    uint4 raw[VEC && sizeof(T) > 1 ? kWords : 1];
    T one[VEC ? 1 : 8];
    __device__ __forceinline__ void load(const T* row, int first, int cols) {
        if constexpr (VEC) {
            if (first < cols) {
                if constexpr (sizeof(T) == 4) {
                    uint32_t w[8];
                    load_32_bytes<true>(row + first, w);
                    raw[0] = make_uint4(w[0], w[1], w[2], w[3]), raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
                } else {
                    raw[0] = __ldcs(reinterpret_cast<const uint4*>(row + first));
                }
            } else {
#pragma unroll
                for (int k = 0; k < kWords; k++) raw[k] = make_uint4(0, 0, 0, 0);
            }
        } else {
            const T* at = row + first;
            if (whole_eight(first, cols)) {
#pragma unroll
                for (int k = 0; k < 8; k++) one[k] = __ldcs(at + 32 * k);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) one[k] = first + 32 * k < cols ? __ldcs(at + 32 * k) : from_float<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = to_float(one[k]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                v[4 * k] = __uint_as_float(raw[k].x), v[4 * k + 1] = __uint_as_float(raw[k].y), v[4 * k + 2] = __uint_as_float(raw[k].z), v[4 * k + 3] = __uint_as_float(raw[k].w);
        } else {
            const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
            for (int k = 0; k < 4; k++) unpack2<T>(w[k], v[2 * k], v[2 * k + 1]);
        }
    }
};
template <bool VEC>
__device__ __forceinline__ void load_weights(const float* w, int first, int cols, float (&v)[8]) {
    if (!w) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = 1.f;
        return;
    }
    if constexpr (VEC) {
        uint32_t u[8] = {};
        if (first < cols) load_32_bytes<false>(w + first, u);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = __uint_as_float(u[k]);
    } else {
        const float* at = w + first;
        if (whole_eight(first, cols)) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = __ldg(at + 32 * k);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = first + 32 * k < cols ? __ldg(at + 32 * k) : 0.f;
        }
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_eight(T* row, int first, int cols, const float (&v)[8]) {
    if constexpr (!VEC) {
        T* at = row + first;
        if (whole_eight(first, cols)) {
#pragma unroll
            for (int k = 0; k < 8; k++) at[32 * k] = from_float<T>(v[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (first + 32 * k < cols) at[32 * k] = from_float<T>(v[k]);
        }
    } else if (first < cols) {
        uint4* at = reinterpret_cast<uint4*>(row + first);
        if constexpr (sizeof(T) == 4) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])),
                         "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])),
                         "r"(__float_as_uint(v[7]))
                         : "memory");
        } else {
            at[0] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
    }
}
template <bool VEC>
__device__ __forceinline__ void store_typed(void* at, int64_t row_at, int type, int first, int cols, const float (&v)[8]) {
    if (type == B200_TYPE_F32)
        store_eight<VEC>(static_cast<float*>(at) + row_at, first, cols, v);
    else if (type == B200_TYPE_BF16)
        store_eight<VEC>(static_cast<bf16*>(at) + row_at, first, cols, v);
    else
        store_eight<VEC>(static_cast<f16*>(at) + row_at, first, cols, v);
}
// Elements of a row on their way to codes: what an activation's outputs have to keep.  Those above 0 and below the smallest code's
// value are moved to that, those between the last code below 1 and 1 to that code's value, which is 1 - 2^-4 up to scales of 2^5 (at
// 2^6 one is the smallest normal code, and the code below it 1 - 2^-3); then the nearest code is the one that is wanted.  Magnitudes
// are in the order of their bits: less 1, what is not to move below the least is 0, the largest of all; less 1's bits, what is below 1
// comes last.  (131072 x 2048 bf16 outputs of CReLU with comparisons and selections 185 us, with these additions in front of maxima and
// minima 161, in a kernel of its own 134.)
__device__ __forceinline__ bool moves_outputs(uint32_t scale) { return scale >= 10u << 23 && scale <= 132u << 23; }
__device__ __forceinline__ uint32_t least_bits(uint32_t scale) { return scale - (9u << 23); }
__device__ __forceinline__ float moved_output(float v, uint32_t least, int act) {
    uint32_t s = __viaddmax_u32(__float_as_uint(v), 0xffffffffu, least - 1u);
    if (act == B200_ACT_RELU) return __uint_as_float(s + 1u);
    s = __viaddmin_u32(s, 1u - 0x3f800000u, 0x3f700000u - 0x3f800000u);
    return __uint_as_float(s + 0x3f800000u);
}
__device__ __forceinline__ uint32_t moved_outputs2(uint32_t w, uint32_t least, int act) {  // two bf16; `least`: in both halves
    uint32_t s = __viaddmax_u16x2(w, 0xffffffffu, least - 0x00010001u);
    if (act == B200_ACT_RELU) return __viaddmin_u16x2(s, 0x00010001u, 0xffffffffu);
    s = __viaddmin_u16x2(s, 0xc081c081u, 0xfff0fff0u);
    return __viaddmin_u16x2(s, 0x3f803f80u, 0xffffffffu);
}
// (v - v is 0, or NaN for what is not finite, which the code is then)
__device__ __forceinline__ uint32_t two_codes(float a, float b, float by_a, float by_b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(fmaf(a, by_a, a - a), fmaf(b, by_b, b - b)), __NV_SATFINITE, __NV_E4M3);
}
// (one call for eight: their code stands beside that of the kernels' usual way otherwise, which then misses the instruction cache)
static __device__ __noinline__ uint2 codes_slowly(float v0, float v1, float v2, float v3, float v4, float v5, float v6, float v7, uint32_t scale, int act) {
    const float v[8] = {v0, v1, v2, v3, v4, v5, v6, v7};
    uint32_t q[8];
#pragma unroll
    for (int k = 0; k < 8; k++) q[k] = code_of_output(v[k], scale, act);
    return make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
}
// Eight codes, as q[k] two each: where the scale is a usual one, else slowly.
template <bool MOVES>
__device__ __forceinline__ bool usual_scale(uint32_t scale) { return scale != kTopScale && (!MOVES || moves_outputs(scale)); }
template <bool MOVES>
__device__ __forceinline__ void eight_codes(const float (&v)[8], uint32_t scale, bool usual, int act, uint32_t (&q)[4]) {
    if (__builtin_expect(usual, 1)) {
        const float by = one_over_scale(scale);
        const uint32_t least = least_bits(scale);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (MOVES)
                q[k] = two_codes(moved_output(v[2 * k], least, act), moved_output(v[2 * k + 1], least, act), by, by);
            else
                q[k] = two_codes(v[2 * k], v[2 * k + 1], by, by);
        }
    } else {
        const uint2 u = codes_slowly(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], scale, act);
        q[0] = u.x & 0xffffu, q[1] = u.x >> 16, q[2] = u.y & 0xffffu, q[3] = u.y >> 16;
    }
}
template <bool VEC>
__device__ __forceinline__ void put_codes(uint8_t* row, int first, int cols, const uint32_t (&q)[4]) {
    if constexpr (VEC) {
        if (first < cols) *reinterpret_cast<uint2*>(row + first) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    } else {
        uint8_t* at = row + first;
        if (whole_eight(first, cols)) {
#pragma unroll
            for (int k = 0; k < 8; k++) at[32 * k] = (uint8_t)(q[k / 2] >> 8 * (k & 1));
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (first + 32 * k < cols) at[32 * k] = (uint8_t)(q[k / 2] >> 8 * (k & 1));
        }
    }
}

// This thread's row and first elements.
struct RowPlace {
    int64_t row;
    bool leader;  // one thread of the row
    int lane_at, step, warps;  // columns lane_at + step * j, j < NV, are its vectors' first
    template <bool VEC, bool SEVERAL = false>
    __device__ __forceinline__ static RowPlace here(int warps) {
        RowPlace p;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        p.warps = warps;
        p.step = 256 * warps;
        if constexpr (!SEVERAL) {  // (no divisions, which cost a short kernel 6 %)
            p.row = warps == 1 ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : (int64_t)blockIdx.x;
            p.leader = lane == 0 && (warps == 1 || warp == 0);
            p.lane_at = (warps == 1 ? 0 : 256 * warp) + (VEC ? 8 * lane : lane);
            return p;
        }
        p.row = (int64_t)blockIdx.x * ((blockDim.x >> 5) / warps) + warp / warps;
        p.leader = lane == 0 && warp % warps == 0;
        p.lane_at = 256 * (warp % warps) + (VEC ? 8 * lane : lane);
        return p;
    }
};

// 1 / sqrt(mean), and what its rounding to fp32 leaves of it: a Newton step from the rounded root, with its error in 64 bits.
__device__ __forceinline__ float root_of_mean(double mean, float& rest) {
    const float first = 1.f / sqrtf((float)mean);
    const float error = (float)fma(-mean * (double)first, (double)first, 1.0);
    const float by = first * 0.5f * error, rstd = first + by;
    const bool fine = finite(rstd) && finite(by);
    rest = fine ? by - (rstd - first) : 0.f;
    return fine ? rstd : first;
}
// t * rstd * w in fp32 may round onto a halfway point of two codes or across it: one code in 10^6 came out as its neighbour.  A
// product within two units of one (bits 19 to 0 of the significand near 0x80000) is formed again: the fp32 number next to the exact one
// towards 0, with its last bit set where it is not exact itself, so that it lies on the right side.  So the roundings of rstd and of both
// products move no code.  What still may: the sum of squares, which is an fp32 sum, and all of them for codes below the smallest
// normal one (2^-6 of the scale), whose halfway points lie elsewhere.  100 M codes of fp32 rows of 2048: 18 neighbours of the nearest,
// without this 60; 16384 of those rows 37.6 us, without this 33.8.
__device__ __forceinline__ bool near_halfway(float y) { return (__float_as_uint(y) - 0x7fffeu) * 4096u < 5u * 4096u; }
template <class TX>
static __device__ __noinline__ float exact_for_code(const TX* x, const TX* residual, const float* weight, float rstd, float rest) {
    const float t = residual ? to_float(*x) + to_float(*residual) : to_float(*x), w = weight ? *weight : 1.f;
    const float n = t * rstd, n_rest = fmaf(t, rest, fmaf(t, rstd, -n)), y = n * w;
    const float y_rest = fmaf(n_rest, w, fmaf(n, w, -y));
    const uint32_t bits = __float_as_uint(y), opposite = (bits ^ __float_as_uint(y_rest)) >> 31;
    return y_rest != 0.f && finite(y_rest) ? __uint_as_float((bits - opposite) | 1u) : y;
}

template <class TX, int NV, bool VEC, bool CODES>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_kernel(b200_rms_norm_op a, int warps, double one_over_cols) {
    __shared__ float sums[kRowWarpsMost];
    __shared__ uint32_t largest[2][kRowWarpsMost];
    const RowPlace p = RowPlace::here<VEC>(warps);
    if (p.row >= a.rows) return;  // (all warps of a row)
    Eight<VEC, TX> x[NV], r[NV];
    const TX* xr = static_cast<const TX*>(a.x) + p.row * a.ldx;
#pragma unroll
    for (int j = 0; j < NV; j++) x[j].load(xr, p.lane_at + p.step * j, a.cols);
    if (a.residual) {
        const TX* rr = static_cast<const TX*>(a.residual) + p.row * a.ldr;
#pragma unroll
        for (int j = 0; j < NV; j++) r[j].load(rr, p.lane_at + p.step * j, a.cols);
    }
    float v[NV][8], squares = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        x[j].get(v[j]);
        if (a.residual) {
            float s[8];
            r[j].get(s);
#pragma unroll
            for (int k = 0; k < 8; k++) v[j][k] += s[k];
        }
        if (a.sum) store_eight<VEC>(static_cast<TX*>(a.sum) + p.row * a.lds, p.lane_at + p.step * j, a.cols, v[j]);
#pragma unroll
        for (int k = 0; k < 8; k++) squares = fmaf(v[j][k], v[j][k], squares);
    }
    float rest;
    const float rstd = root_of_mean((double)row_sum(squares, warps, sums) * one_over_cols + (double)a.eps, rest);
    if (a.rstd && p.leader) a.rstd[p.row] = rstd;
    float most = 0.f;  // (NaN, which no scale is to know of, loses against every number)
#pragma unroll
    for (int j = 0; j < NV; j++) {
        float w[8];
        load_weights<VEC>(a.weight, p.lane_at + p.step * j, a.cols, w);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            v[j][k] = v[j][k] * rstd * w[k];
            if constexpr (CODES) most = fmaxf(most, fabsf(v[j][k]));
        }
        if constexpr (!CODES) store_typed<VEC>(a.y, p.row * a.ldy, a.y_type, p.lane_at + p.step * j, a.cols, v[j]);
    }
    if constexpr (CODES) {
        uint32_t m = row_max(magnitude_bits(most), warps, largest[0]);
        if (m >= 0x7f800000u) {  // the same in all threads of the row
            m = 0;
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int k = 0; k < 8; k++) m = max(m, finite_magnitude(v[j][k]));
            m = row_max(m, warps, largest[1]);
        }
        const uint32_t scale = scale_bits(m);
        const bool usual = usual_scale<false>(scale);
        if (p.leader) a.scale[p.row] = __uint_as_float(scale);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            uint32_t past = 0xffffffffu;
#pragma unroll
            for (int k = 0; k < 8; k++) past = __viaddmin_u32(__float_as_uint(v[j][k]) << 12, 0u - (0x7fffeu << 12), past);
            if (past < 5u << 12) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int c = p.lane_at + p.step * j + (VEC ? k : 32 * k);
                    if (near_halfway(v[j][k]) && c < a.cols)
                        v[j][k] = exact_for_code(xr + c, a.residual ? static_cast<const TX*>(a.residual) + p.row * a.ldr + c : nullptr, a.weight ? a.weight + c : nullptr, rstd, rest);
                }
            }
            uint32_t q[4];
            eight_codes<false>(v[j], scale, usual, B200_ACT_NONE, q);
            put_codes<VEC>(static_cast<uint8_t*>(a.y) + p.row * a.ldy, p.lane_at + p.step * j, a.cols, q);
        }
    }
}

// Elements of 16 bits are compared two at a time: one by one the ALU pipe takes longer than HBM (131072 rows of 2048 bf16 outputs of
// CReLU 207 us, so 134, for 805 MB; plain values 120).
// OUTPUTS: of an activation.
template <class TX, int NV, bool VEC, bool OUTPUTS>
static __global__ void __launch_bounds__(kRowThreads) pack8_rows_kernel(b200_pack8_op a, int warps) {
    constexpr bool TWO = VEC && sizeof(TX) == 2;
    __shared__ uint32_t largest[2][kRowWarpsMost];
    const RowPlace p = RowPlace::here<VEC>(warps);
    if (p.row >= a.rows) return;
    Eight<VEC, TX> x[NV];
    const TX* xr = static_cast<const TX*>(a.x) + p.row * a.ldx;
#pragma unroll
    for (int j = 0; j < NV; j++) x[j].load(xr, p.lane_at + p.step * j, a.cols);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if constexpr (TWO) {  // magnitudes are in the order of their bits
            m = __vmaxu2(m, x[j].raw[0].x & 0x7fff7fffu);
            m = __vmaxu2(m, x[j].raw[0].y & 0x7fff7fffu);
            m = __vmaxu2(m, x[j].raw[0].z & 0x7fff7fffu);
            m = __vmaxu2(m, x[j].raw[0].w & 0x7fff7fffu);
        } else {
            float v[8];
            x[j].get(v);
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, magnitude_bits(v[k]));
        }
    }
    if constexpr (TWO) {
        float low, high;
        unpack2<TX>(m, low, high);
        m = max(magnitude_bits(low), magnitude_bits(high));
    }
    m = row_max(m, warps, largest[0]);
    if (m >= 0x7f800000u) {
        m = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float v[8];
            x[j].get(v);
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, finite_magnitude(v[k]));
        }
        m = row_max(m, warps, largest[1]);
    }
    const uint32_t scale = scale_bits(m);
    if (p.leader) a.scale[p.row] = __uint_as_float(scale);
    const bool usual = usual_scale<OUTPUTS>(scale);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        constexpr bool kTwoMoved = OUTPUTS && TWO && std::is_same<TX, bf16>::value;
        uint32_t q[4];
        float v[8];
        if (kTwoMoved && usual) {
            const uint32_t least = (least_bits(scale) >> 16) * 0x00010001u;
            uint4& w = x[j].raw[0];
            w = make_uint4(moved_outputs2(w.x, least, a.act), moved_outputs2(w.y, least, a.act), moved_outputs2(w.z, least, a.act), moved_outputs2(w.w, least, a.act));
        }
        x[j].get(v);
        eight_codes<OUTPUTS && !kTwoMoved>(v, scale, usual, a.act, q);
        put_codes<VEC>(static_cast<uint8_t*>(a.q) + p.row * a.ldq, p.lane_at + p.step * j, a.cols, q);
    }
}

// The gradient.  A group of W warps takes rows group, group + groups, ...; dy * n of its columns is added up in registers over
// its rows, and the CTA's groups in shared memory at the end: parts[CTA][cols].
template <class TX, class TD, int NV, bool VEC>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_backward_kernel(b200_rms_norm_grad_op a, float* parts, int warps) {
    extern __shared__ float added[];  // [groups of the CTA][cols], where there are several
    __shared__ float sums[2][kRowWarpsMost];
    const RowPlace p = RowPlace::here<VEC, true>(warps);
    const int groups = (blockDim.x >> 5) / warps, group = (threadIdx.x >> 5) / warps;
    step_begin(nullptr);
    float dw[NV][8] = {};
    int turn = 0;
    const bool through = a.dsum && a.dx;
    const int64_t stride = (int64_t)gridDim.x * groups;
    Eight<VEC, TX> s[NV], ds[NV];
    Eight<VEC, TD> dy[NV];
    float rstd = 0.f;
    auto fetch = [&](int64_t row) {
        const TX* sr = static_cast<const TX*>(a.sum) + row * a.lds;
        const TD* dr = static_cast<const TD*>(a.dy) + row * a.lddy;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            s[j].load(sr, p.lane_at + p.step * j, a.cols);
            dy[j].load(dr, p.lane_at + p.step * j, a.cols);
        }
        if (through) {
            const TX* dsr = static_cast<const TX*>(a.dsum) + row * a.ldds;
#pragma unroll
            for (int j = 0; j < NV; j++) ds[j].load(dsr, p.lane_at + p.step * j, a.cols);
        }
        rstd = a.rstd[row];
    };
    // The next row's loads go out before this one's sum and stores where there are registers for that: 131072 x 2048 bf16 with dsum 397 us
    // without, 333 with; in fp32, with half as many warps on an SM then, 490 and 565.
    constexpr bool kAhead = VEC && NV <= 2 && sizeof(TX) == 2 && sizeof(TD) == 2;
    if (kAhead && p.row < a.rows) fetch(p.row);
    for (int64_t row = p.row; row < a.rows; row += stride, turn ^= 1) {
        if (!kAhead) fetch(row);
        float n[NV][8], g[NV][8], d[NV][8], dot = 0.f;
        const float by = rstd;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float w[8];
            load_weights<VEC>(a.weight, p.lane_at + p.step * j, a.cols, w);
            s[j].get(n[j]);
            dy[j].get(g[j]);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                n[j][k] *= by;  // (past the columns 0; NaN where rstd is infinite, as all of the row's dx is then)
                dw[j][k] = fmaf(g[j][k], n[j][k], dw[j][k]);
                g[j][k] *= w[k];
                dot = fmaf(g[j][k], n[j][k], dot);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (through) {
                ds[j].get(d[j]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) d[j][k] = 0.f;
            }
        }
        if (kAhead && row + stride < a.rows) fetch(row + stride);
        if (!a.dx) continue;
        const float mean = row_sum<true>(dot, warps, sums[turn]) / (float)a.cols;
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int k = 0; k < 8; k++) d[j][k] = fmaf(by, fmaf(-n[j][k], mean, g[j][k]), d[j][k]);
            store_eight<VEC>(static_cast<TX*>(a.dx) + row * a.lddx, p.lane_at + p.step * j, a.cols, d[j]);
        }
    }
    if (!a.dweight) return;
    float* part = parts + (int64_t)blockIdx.x * a.cols;
    float* to = groups == 1 ? part : added + (int64_t)group * a.cols;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int c = p.lane_at + p.step * j + (VEC ? k : 32 * k);
            if (c < a.cols) to[c] = dw[j][k];
        }
    if (groups == 1) return;
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float v = 0.f;
        for (int k = 0; k < groups; k++) v += added[(int64_t)k * a.cols + c];
        part[c] = v;
    }
}

// out[c] = the sum of parts[...][c]: 32 columns a CTA, 32 warps that take every 32nd part.
constexpr int kAddThreads = 1024;
static __global__ void __launch_bounds__(kAddThreads) add_parts_kernel(const float* parts, int n_parts, int cols, float* out) {
    __shared__ float sums[32][33];
    step_waits();
    if (threadIdx.x == 0) step_hands_on();  // (products of the same call may start beside it)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int k = warp; k < n_parts; k += 32) v += __ldcg(parts + (int64_t)k * cols + c);
    }
    sums[lane][warp] = v;
    __syncthreads();
    v = warp_sum(sums[warp][lane]);  // a warp per column
    if (lane == 0 && blockIdx.x * 32 + warp < cols) out[blockIdx.x * 32 + warp] = v;
}

// ---- rows of any length: a CTA of eight warps per row, element by element (a norm's codes are those of its fp32 products here)

__device__ __forceinline__ float cta_sum(float v, float* shared) {
    v = row_sum(v, kRowWarpsMost, shared);
    __syncthreads();
    return v;
}
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* shared) {
    v = row_max(v, kRowWarpsMost, shared);
    __syncthreads();
    return v;
}

template <class TX>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_any_kernel(b200_rms_norm_op a) {
    __shared__ float sums[kRowWarpsMost];
    __shared__ uint32_t largest[kRowWarpsMost];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
        const TX* r = a.residual ? static_cast<const TX*>(a.residual) + row * a.ldr : nullptr;
        auto total = [&](int c) { return r ? to_float(x[c]) + to_float(r[c]) : to_float(x[c]); };
        float v = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
            const float t = total(c);
            v = fmaf(t, t, v);
            if (a.sum) static_cast<TX*>(a.sum)[row * a.lds + c] = from_float<TX>(t);
        }
        const float rstd = 1.f / sqrtf(cta_sum(v, sums) / (float)a.cols + a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
        auto normed = [&](int c) { return total(c) * rstd * (a.weight ? a.weight[c] : 1.f); };
        if (a.y_type == B200_TYPE_E4M3) {
            uint32_t m = 0;
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) m = max(m, finite_magnitude(normed(c)));
            const uint32_t scale = scale_bits(cta_max(m, largest));
            if (threadIdx.x == 0) a.scale[row] = __uint_as_float(scale);
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) static_cast<uint8_t*>(a.y)[row * a.ldy + c] = code_of_output(normed(c), scale, B200_ACT_NONE);
        } else {
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) store_value(a.y, row * a.ldy + c, a.y_type, normed(c));
        }
    }
}
template <class TX, class TD>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_dx_any_kernel(b200_rms_norm_grad_op a) {
    __shared__ float sums[kRowWarpsMost];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* s = static_cast<const TX*>(a.sum) + row * a.lds;
        const TD* dy = static_cast<const TD*>(a.dy) + row * a.lddy;
        const TX* ds = a.dsum ? static_cast<const TX*>(a.dsum) + row * a.ldds : nullptr;
        const float rstd = a.rstd[row];
        auto g = [&](int c) { return to_float(dy[c]) * (a.weight ? a.weight[c] : 1.f); };
        float v = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) v = fmaf(g(c), to_float(s[c]) * rstd, v);
        const float mean = cta_sum(v, sums) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
            const float dx = rstd * (g(c) - to_float(s[c]) * rstd * mean);
            static_cast<TX*>(a.dx)[row * a.lddx + c] = from_float<TX>(ds ? dx + to_float(ds[c]) : dx);
        }
    }
}
// Sums over a piece of the rows, a thread per column: parts[piece][cols].
template <class TX, class TD>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_dweight_any_kernel(b200_rms_norm_grad_op a, float* parts) {
    const int c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    float v = 0.f;
    for (int64_t row = first; row < last; row++)
        v = fmaf(to_float(static_cast<const TD*>(a.dy)[row * a.lddy + c]), to_float(static_cast<const TX*>(a.sum)[row * a.lds + c]) * a.rstd[row], v);
    parts[(int64_t)blockIdx.y * a.cols + c] = v;
}
template <class TX>
static __global__ void __launch_bounds__(kRowThreads) pack8_rows_any_kernel(b200_pack8_op a) {
    __shared__ uint32_t largest[kRowWarpsMost];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
        uint32_t m = 0;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) m = max(m, finite_magnitude(to_float(x[c])));
        const uint32_t scale = scale_bits(cta_max(m, largest));
        if (threadIdx.x == 0) a.scale[row] = __uint_as_float(scale);
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads)
            static_cast<uint8_t*>(a.q)[row * a.ldq + c] = code_of_output(to_float(x[c]), scale, a.act);
    }
}

// ---- by column

// A thread takes V columns (eight side by side, or one) of the rows of its CTA's piece, the CTA's threads `across` of them side by
// side and the rest in other rows.  Scales are in the order of their bits and none is 0, so the largest of the pieces' is the
// column's; a column without a finite value but 0 is left at 0, which pack8_columns_kernel takes for 1 and whose first piece
// writes 1 there: the others take either as 1.
struct ColumnPlace {
    int column;
    int64_t row, last, step;
    __device__ __forceinline__ ColumnPlace(int rows, int across, int v) {
        const int64_t first = (int64_t)rows * blockIdx.y / gridDim.y;
        last = (int64_t)rows * (blockIdx.y + 1) / gridDim.y;
        column = (blockIdx.x * across + (int)threadIdx.x % across) * v;
        step = kRowThreads / across;
        row = first + (int)threadIdx.x / across;
    }
};
constexpr int kColumnRows = 4;  // in flight
template <class T>
__device__ __forceinline__ void load_columns(const T* at, float (&v)[8]) {
    Eight<true, T> e;
    e.load(at, 0, 8);
    e.get(v);
}
template <class T>
__device__ __forceinline__ void load_columns(const T* at, float (&v)[1]) {
    v[0] = to_float(*at);
}
template <class TX, int V>
static __global__ void __launch_bounds__(kRowThreads) column_scales_kernel(b200_pack8_op a, int across) {
    __shared__ uint32_t largest[kRowThreads * V];
    ColumnPlace p(a.rows, across, V);
    uint32_t m[V] = {};
    const TX* x = static_cast<const TX*>(a.x) + p.column;
    if (p.column < a.cols)
        for (; p.row < p.last; p.row += p.step * kColumnRows) {
            float v[kColumnRows][V];
#pragma unroll
            for (int r = 0; r < kColumnRows; r++) load_columns(x + min(p.row + r * p.step, p.last - 1) * a.ldx, v[r]);
#pragma unroll
            for (int r = 0; r < kColumnRows; r++)
#pragma unroll
                for (int k = 0; k < V; k++) m[k] = max(m[k], finite_magnitude(v[r][k]));
        }
    // one word per column and CTA: atomics of all threads took most of the time (65536 x 512 bf16: 430 us)
#pragma unroll
    for (int k = 0; k < V; k++) largest[k * kRowThreads + threadIdx.x] = m[k];
    __syncthreads();
    for (int c = threadIdx.x; c < across * V; c += kRowThreads) {
        const int column = blockIdx.x * across * V + c;
        uint32_t most = 0;
        for (int r = 0; r < kRowThreads / across; r++) most = max(most, largest[c % V * kRowThreads + r * across + c / V]);
        if (column < a.cols && most) atomicMax(reinterpret_cast<uint32_t*>(a.scale) + column, scale_bits(most));
    }
}
template <class TX, int V>
static __global__ void __launch_bounds__(kRowThreads) pack8_columns_kernel(b200_pack8_op a, int across) {
    ColumnPlace p(a.rows, across, V);
    if (p.column >= a.cols) return;
    uint32_t scale[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        volatile uint32_t* at = reinterpret_cast<uint32_t*>(a.scale) + p.column + k;
        scale[k] = *at;
        if (scale[k] == 0) {
            scale[k] = scale_bits(0);
            if (blockIdx.y == 0) *at = scale[k];
        }
    }
    bool quick = true;
    float by[V];
#pragma unroll
    for (int k = 0; k < V; k++) by[k] = one_over_scale(scale[k]);
#pragma unroll
    for (int k = 0; k < V; k++) quick &= scale[k] != kTopScale && (a.act == B200_ACT_NONE || moves_outputs(scale[k]));
    const TX* x = static_cast<const TX*>(a.x) + p.column;
    uint8_t* q = static_cast<uint8_t*>(a.q) + p.column;
    for (; p.row < p.last; p.row += p.step * kColumnRows) {
        float v[kColumnRows][V];
#pragma unroll
        for (int r = 0; r < kColumnRows; r++) load_columns(x + min(p.row + r * p.step, p.last - 1) * a.ldx, v[r]);
#pragma unroll
        for (int r = 0; r < kColumnRows; r++) {
            if (p.row + r * p.step >= p.last) break;
            uint32_t code[V];
            if (quick) {
                if (a.act != B200_ACT_NONE)
#pragma unroll
                    for (int k = 0; k < V; k++) v[r][k] = moved_output(v[r][k], least_bits(scale[k]), a.act);
#pragma unroll
                for (int k = 0; k < V; k += 2) {
                    constexpr int kNext = V > 1 ? 1 : 0;
                    const uint32_t two = two_codes(v[r][k], v[r][k + kNext], by[k], by[k + kNext]);
                    code[k + kNext] = two >> 8;
                    code[k] = two & 0xffu;
                }
            } else {
#pragma unroll
                for (int k = 0; k < V; k++) code[k] = code_of_output(v[r][k], scale[k], a.act);
            }
            if constexpr (V == 8)
                *reinterpret_cast<uint2*>(q + (p.row + r * p.step) * a.ldq) = make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
                                                                                        code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
            else
                q[(p.row + r * p.step) * a.ldq] = (uint8_t)code[0];
        }
    }
}

// ---- codes to values: the threads of a CTA `across` side by side, V codes each (sixteen, eight or one), kUnpackRows rows in flight
constexpr int kUnpackRows = 4;
template <class TY, int V>
static __global__ void __launch_bounds__(kRowThreads) unpack8_kernel(b200_unpack8_op a, int across) {
    const int rows_at_once = kRowThreads / across, lane = (int)threadIdx.x % across;
    const int64_t first = (int64_t)blockIdx.x * rows_at_once * kUnpackRows + (int)threadIdx.x / across;
    const uint8_t* q = static_cast<const uint8_t*>(a.q);
    for (int c = lane * V; c < a.cols; c += across * V) {
        uint4 code[kUnpackRows];
        float scale[kUnpackRows];
#pragma unroll
        for (int r = 0; r < kUnpackRows; r++) {
            const int64_t row = min(first + (int64_t)r * rows_at_once, (int64_t)a.rows - 1);
            if constexpr (V == 16) {
                code[r] = __ldcs(reinterpret_cast<const uint4*>(q + row * a.ldq + c));
            } else if constexpr (V == 8) {
                const uint2 w = __ldcs(reinterpret_cast<const uint2*>(q + row * a.ldq + c));
                code[r].x = w.x, code[r].y = w.y;
            } else
                code[r].x = q[row * a.ldq + c];
            scale[r] = a.by_column ? 1.f : __ldg(a.scale + row);
        }
#pragma unroll
        for (int r = 0; r < kUnpackRows; r++) {
            const int64_t row = first + (int64_t)r * rows_at_once;
            if (row >= a.rows) break;
            TY* y = static_cast<TY*>(a.y) + row * a.ldy + c;
            if constexpr (V > 1) {
                const uint32_t w[4] = {code[r].x, code[r].y, code[r].z, code[r].w};
#pragma unroll
                for (int h = 0; h < V / 8; h++) {
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        const uint32_t pair = w[2 * h + k / 4] >> 8 * (k & 3);
                        const __half2_raw halves = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
                        const float2 f = __half22float2(__half2(halves));
                        v[k] = f.x * (a.by_column ? __ldg(a.scale + c + 8 * h + k) : scale[r]);
                        v[k + 1] = f.y * (a.by_column ? __ldg(a.scale + c + 8 * h + k + 1) : scale[r]);
                    }
                    store_eight<true>(y, 8 * h, 16, v);
                }
            } else {
                *y = from_float<TY>(to_float(e4m3{(uint8_t)code[r].x}) * (a.by_column ? __ldg(a.scale + c) : scale[r]));
            }
        }
    }
}

}  // namespace b200
