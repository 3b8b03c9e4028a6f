// Matrices in 4 bits: codes and scales made, turned back, and the dense layer of a few rows on them.
//
// A code is e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.  32 elements along the axis that a product sums over are a group and
// share a power of two as scale, a byte that holds its exponent + 127 (255: NaN, and so is the group).  A row of codes is whole groups of 16
// bytes, the even element of a pair in a byte's low half.  Scales lie in tiles of 128 rows by four groups, as the tensor pipe takes them
// (FourScales): a tile's 512 bytes are one copy into shared memory and one from there into tensor memory.
#pragma once
#include <cuda_runtime.h>

#include <cstring>

#include "launch.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kFourThreads = 256;

struct FourScales {
    int64_t groups;  // of a row
    __host__ __device__ int64_t across() const { return (groups + 3) / 4; }
    __host__ __device__ int64_t at(int64_t row, int64_t group) const {
        return ((row >> 7) * across() + (group >> 2)) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4 + (group & 3);
    }
};

// The scale's byte for a largest magnitude given by its bits: the smallest power of two from 2^-126 on with magnitude / scale <= 6 = 1.5 *
// 2^2; 2^0 for a magnitude of 0, NaN for one that is not finite.
__device__ __forceinline__ uint32_t four_scale(uint32_t magnitude) {
    if (magnitude >= 0x7f800000u) return 255;
    if (magnitude == 0) return 127;
    return (uint32_t)max((int)(magnitude >> 23) - 2 + ((magnitude & 0x7fffffu) > 0x400000u), 1);
}
// 1 / scale for a byte that four_scale made
__device__ __forceinline__ float four_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }
__device__ __forceinline__ float four_value(uint32_t scale) {
    return __uint_as_float(scale == 255 ? 0x7fffffffu : scale ? scale << 23 : 0x400000u);
}
// Eight codes of values that are scaled already: nearest, halves to the even one.
__device__ __forceinline__ uint32_t four_codes(const float (&v)[8]) {
    uint32_t w;
    asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\ncvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\nmov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}
// Eight values (exact in 16 bits) of codes.
__device__ __forceinline__ void four_values(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int k = 0; k < 4; k++) unpack2<f16>(h[k], v[2 * k], v[2 * k + 1]);
}
// Codes of a group's eight values at the group's scale.  At the largest scale, 2^126, a value that would round up out of fp32 rounds down.
__device__ __forceinline__ uint32_t four_codes_at(float (&v)[8], uint32_t scale) {
    if (scale == 255) return 0;
    const float f = four_inverse(scale);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] *= f;
    if (__builtin_expect(scale == 253, 0)) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = fminf(fmaxf(v[k], -3.f), 3.f);
    }
    return four_codes(v);
}

// A place in a matrix of `width` places a row that moves on by the same number of places each time.
struct Place {
    uint32_t row, at, rows_on, on, width;
    __device__ Place(uint32_t first, uint32_t step, uint32_t width_) : row(first / width_), at(first % width_), rows_on(step / width_), on(step % width_), width(width_) {}
    __device__ __forceinline__ void next() {
        row += rows_on, at += on;
        if (at >= width) at -= width, row++;
    }
};

// WAY: how a thread's elements of a row lie: 2, sixteen together on 32 bytes; 1, eight on 16; 0, eight anywhere.
template <int WAY>
constexpr int kFourEach = WAY == 2 ? 16 : 8;
// Those from `first` on; what lies at or past `cols` is 0.
template <int WAY, class T>
__device__ __forceinline__ void load_elements(const T* row, int64_t first, int64_t cols, T (&v)[kFourEach<WAY>]) {
    constexpr int kBytes = kFourEach<WAY> * sizeof(T);
    if constexpr (WAY == 2) {
        uint32_t w[kBytes / 4] = {};
        if (first < cols)
#pragma unroll
            for (int k = 0; k < kBytes / 32; k++)
                asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[8 * k]), "=r"(w[8 * k + 1]), "=r"(w[8 * k + 2]), "=r"(w[8 * k + 3]), "=r"(w[8 * k + 4]), "=r"(w[8 * k + 5]), "=r"(w[8 * k + 6]), "=r"(w[8 * k + 7])
                             : "l"(reinterpret_cast<const unsigned char*>(row + first) + 32 * k));
        memcpy(v, w, kBytes);
    } else if constexpr (WAY == 1) {
        uint4 w[kBytes / 16] = {};
        if (first < cols)
#pragma unroll
            for (int k = 0; k < kBytes / 16; k++) w[k] = __ldcs(reinterpret_cast<const uint4*>(row + first) + k);
        memcpy(v, w, kBytes);
    } else {
#pragma unroll
        for (int k = 0; k < kFourEach<WAY>; k++) v[k] = first + k < cols ? __ldcs(row + first + k) : from_float<T>(0.f);
    }
}
// The largest magnitude of N elements, as the bits of fp32.
template <class T, int N>
__device__ __forceinline__ uint32_t most_of(const T (&v)[N]) {
    uint32_t most = 0;
    if constexpr (sizeof(T) == 2) {  // two at a time: magnitudes are in the order of their bits
        uint32_t w[N / 2];
        memcpy(w, v, sizeof(v));
#pragma unroll
        for (int k = 0; k < N / 2; k++) most = __vmaxu2(most, w[k] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
        const uint16_t bits = (uint16_t)most;
        T largest;
        memcpy(&largest, &bits, 2);
        return __float_as_uint(to_float(largest)) & 0x7fffffffu;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) most = max(most, __float_as_uint(v[k]) & 0x7fffffffu);
        return most;
    }
}

// Rows to codes: a group's elements lie in two or four neighbouring threads, kFourAhead places of a thread are on their way.  Also the scales' bytes past the last
// row and the last group (127).  HBM bound.
constexpr int kFourAhead = 4;
template <class T, int WAY>
static __global__ void __launch_bounds__(kFourThreads) pack4_rows_kernel(b200_pack4_op a, FourScales s) {
    constexpr int kEach = kFourEach<WAY>, kShare = 32 / kEach, kAhead = kEach * sizeof(T) > 32 ? kFourAhead / 2 : kFourAhead;
    const uint32_t rows_all = (uint32_t)((a.rows + 127ll) / 128 * 128);  // (times eight or more places a row: a warp's places are all there or none)
    Place p(blockIdx.x * kFourThreads + threadIdx.x, gridDim.x * kFourThreads, (uint32_t)s.across() * 4 * kShare);
    const T* x = static_cast<const T*>(a.x);
    uint8_t* q = static_cast<uint8_t*>(a.q);
    const uint32_t last = (uint32_t)a.rows - 1, groups = (uint32_t)s.groups;
    while (p.row < rows_all) {
        T in[kAhead][kEach];
        Place ahead = p;
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            load_elements<WAY>(x + min(ahead.row, last) * a.ldx, (int64_t)ahead.at * kEach, a.cols, in[k]);
            ahead.next();
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            if (p.row >= rows_all) return;
            uint32_t most = most_of(in[k]);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            if (kShare == 4) most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const uint32_t group = p.at / kShare;
            const bool here = p.row <= last && group < groups;
            const uint32_t scale = here ? four_scale(most) : 127;
            if (here) {
                uint32_t w[kEach / 8];
#pragma unroll
                for (int h = 0; h < kEach / 8; h++) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = to_float(in[k][8 * h + i]);
                    w[h] = four_codes_at(v, scale);
                }
                uint8_t* to = q + p.row * a.ldq + p.at * (kEach / 2);
                if constexpr (kEach == 16)
                    *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
                else
                    *reinterpret_cast<uint32_t*>(to) = w[0];
            }
            if (p.at % kShare == 0) a.scale[s.at(p.row, group)] = (uint8_t)scale;
            p.next();
        }
    }
}

// Columns to rows of codes: a thread takes 32 elements of a column, a CTA 64 columns by four groups.
template <class T>
static __global__ void __launch_bounds__(kFourThreads) pack4_columns_kernel(b200_pack4_op a, FourScales s) {
    const int64_t column = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    for (int64_t group = blockIdx.y * 4ll + (threadIdx.x >> 6); group < s.across() * 4; group += gridDim.y * 4ll) {
        const bool here = column < a.cols && group < s.groups;
        uint32_t scale = 127;
        if (here) {
            const T* x = static_cast<const T*>(a.x) + group * 32 * a.ldx + column;
            const int there = (int)min((int64_t)32, a.rows - group * 32);
            T in[32];
            if (there == 32) {
#pragma unroll
                for (int k = 0; k < 32; k++) in[k] = __ldcs(x + k * a.ldx);
            } else {
#pragma unroll
                for (int k = 0; k < 32; k++) in[k] = k < there ? __ldcs(x + k * a.ldx) : from_float<T>(0.f);
            }
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < 32; k++) most = max(most, __float_as_uint(to_float(in[k])) & 0x7fffffffu);
            scale = four_scale(most);
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 4; h++) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = to_float(in[8 * h + k]);
                w[h] = four_codes_at(v, scale);
            }
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.q) + column * a.ldq + group * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        a.scale[s.at(column, group)] = (uint8_t)scale;
    }
}

template <bool VEC, class T>
__device__ __forceinline__ void store_values(T* row, int64_t first, int64_t cols, const float (&v)[8]) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(row + first)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(row + first)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4*>(row + first) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (first + k < cols) row[first + k] = from_float<T>(v[k]);
    }
}

// Codes to values: sixteen a thread where rows of values start on 32 bytes, else eight.
template <class T, int WAY>
static __global__ void __launch_bounds__(kFourThreads) unpack4_rows_kernel(b200_unpack4_op a, FourScales s) {
    constexpr int kEach = kFourEach<WAY>;
    Place p(blockIdx.x * kFourThreads + threadIdx.x, gridDim.x * kFourThreads, (uint32_t)((a.cols + kEach - 1ll) / kEach));
    const uint8_t* q = static_cast<const uint8_t*>(a.q);
    const uint32_t rows = (uint32_t)a.rows;
    while (p.row < rows) {
        uint2 code[kFourAhead];
        uint8_t scale[kFourAhead];
        Place ahead = p;
#pragma unroll
        for (int k = 0; k < kFourAhead; k++) {
            const uint32_t row = min(ahead.row, rows - 1);
            const uint8_t* from = q + row * a.ldq + ahead.at * (kEach / 2);
            if constexpr (kEach == 16)
                code[k] = __ldcs(reinterpret_cast<const uint2*>(from));
            else
                code[k].x = __ldcs(reinterpret_cast<const uint32_t*>(from));
            scale[k] = __ldg(a.scale + s.at(row, ahead.at * kEach / 32));
            ahead.next();
        }
#pragma unroll
        for (int k = 0; k < kFourAhead; k++) {
            if (p.row >= rows) return;
            const float f = four_value(scale[k]);
            float v[kEach / 8][8];
#pragma unroll
            for (int h = 0; h < kEach / 8; h++) {
                four_values(h ? code[k].y : code[k].x, v[h]);
#pragma unroll
                for (int i = 0; i < 8; i++) v[h][i] *= f;
            }
            T* y = static_cast<T*>(a.y) + p.row * a.ldy;
            const int64_t first = (int64_t)p.at * kEach;
            if constexpr (WAY == 2) {
                uint32_t w[kEach * sizeof(T) / 4];
#pragma unroll
                for (int i = 0; i < kEach; i += 2) {
                    if constexpr (sizeof(T) == 4)
                        w[i] = __float_as_uint(v[i / 8][i % 8]), w[i + 1] = __float_as_uint(v[i / 8][i % 8 + 1]);
                    else
                        w[i / 2] = pack2<T>(v[i / 8][i % 8], v[i / 8][i % 8 + 1]);
                }
#pragma unroll
                for (int i = 0; i < (int)(kEach * sizeof(T) / 4); i += 8)
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(y + first) + i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                                 "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                                 : "memory");
            } else {
                store_values<WAY == 1>(y, first, a.cols, v[0]);
            }
            p.next();
        }
    }
}
// ... of columns: as pack4_columns_kernel
template <class T>
static __global__ void __launch_bounds__(kFourThreads) unpack4_columns_kernel(b200_unpack4_op a, FourScales s) {
    const int64_t column = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    if (column >= a.cols) return;
    for (int64_t group = blockIdx.y * 4ll + (threadIdx.x >> 6); group < s.groups; group += gridDim.y * 4ll) {
        const uint4 code = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + column * a.ldq + group * 16);
        const float f = four_value(__ldg(a.scale + s.at(column, group)));
        const uint32_t w[4] = {code.x, code.y, code.z, code.w};
        T* y = static_cast<T*>(a.y) + group * 32 * a.ldy + column;
        const int there = (int)min((int64_t)32, a.rows - group * 32);
#pragma unroll
        for (int h = 0; h < 4; h++) {
            float v[8];
            four_values(w[h], v);
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (8 * h + k < there) y[(8 * h + k) * a.ldy] = from_float<T>(v[k] * f);
        }
    }
}

// ---- the dense layer of up to eight rows
//
// Twice a code's value is a whole number of five bits, so a group's 32 products are summed exactly by integer dot products of bytes, and
// the groups' sums, times both scales, in fp32.  W is read once, 16 bytes a lane; a warp takes one output at a time, its lanes the groups.
// The rows' codes are turned into bytes once per CTA.
constexpr int kFewFourRows = 8, kFewFourBytes = 64 * 1024;  // of x as bytes

// Eight codes to twice their values in bytes: elements 0 to 3 and 4 to 7.
__device__ __forceinline__ void four_bytes(uint32_t w, uint32_t& low, uint32_t& high) {
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t four = w >> 16 * h, size = four & 0x7777u, sign = four & 0x8888u;
        const uint32_t above = __byte_perm(0x03020100u, 0x0c080604u, size), below = __byte_perm(0xfdfeff00u, 0xf4f8fafcu, size);
        uint32_t mask;  // (8: the sign of byte 0, all over; 4: byte 4, which is 0)
        asm("prmt.b32 %0, %1, %2, %3;" : "=r"(mask) : "r"(0x80u), "r"(0u), "r"(sign | (sign ^ 0x8888u) >> 1));
        out[h] = (above & ~mask) | (below & mask);
    }
    low = out[0], high = out[1];
}
// v * 2^e for the sum of two scales' exponents
__device__ __forceinline__ float times_power(float v, int e) {
    const int first = min(max(e, -126), 127), rest = max(e - first, -126);
    return v * __uint_as_float((uint32_t)(first + 127) << 23) * __uint_as_float((uint32_t)(rest + 127) << 23);
}

template <int R>
static __global__ void __launch_bounds__(256) dense4_few_kernel(b200_dense4_op a, FourScales s) {
    extern __shared__ uint4 bytes[];  // [R][2][groups]: the halves of a group's 32 bytes
    const int groups = (int)s.groups, lane = threadIdx.x & 31;
    uint8_t* x_scale = reinterpret_cast<uint8_t*>(bytes + 2 * R * groups);
    const uint8_t* w = static_cast<const uint8_t*>(a.w);
    for (int k = threadIdx.x; k < R * groups; k += 256) {
        const int r = k / groups, g = k % groups;
        uint4 code = make_uint4(0, 0, 0, 0);
        uint32_t scale = 127;
        if (r < a.rows) {
            code = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.x) + r * a.ldx + g * 16);
            scale = a.x_scale[s.at(r, g)];
        }
        uint4 b[2];
        four_bytes(code.x, b[0].x, b[0].y);
        four_bytes(code.y, b[0].z, b[0].w);
        four_bytes(code.z, b[1].x, b[1].y);
        four_bytes(code.w, b[1].z, b[1].w);
        bytes[(2 * r) * groups + g] = b[0];
        bytes[(2 * r + 1) * groups + g] = b[1];
        x_scale[k] = (uint8_t)scale;
    }
    __syncthreads();
    for (int64_t n = blockIdx.x * 8ll + (threadIdx.x >> 5); n < a.out; n += gridDim.x * 8ll) {
        float sum[R] = {};
        const uint8_t* row = w + n * a.ldw;
#pragma unroll 4
        for (int g = lane; g < groups; g += 32) {
            const uint4 code = __ldg(reinterpret_cast<const uint4*>(row + g * 16));
            const int w_scale = a.w_scale[s.at(n, g)];
            uint32_t b[8];
            four_bytes(code.x, b[0], b[1]);
            four_bytes(code.y, b[2], b[3]);
            four_bytes(code.z, b[4], b[5]);
            four_bytes(code.w, b[6], b[7]);
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint4 low = bytes[(2 * r) * groups + g], high = bytes[(2 * r + 1) * groups + g];
                int v = __dp4a((int)low.x, (int)b[0], 0);
                v = __dp4a((int)low.y, (int)b[1], v);
                v = __dp4a((int)low.z, (int)b[2], v);
                v = __dp4a((int)low.w, (int)b[3], v);
                v = __dp4a((int)high.x, (int)b[4], v);
                v = __dp4a((int)high.y, (int)b[5], v);
                v = __dp4a((int)high.z, (int)b[6], v);
                v = __dp4a((int)high.w, (int)b[7], v);
                const int own = x_scale[r * groups + g];
                const float f = times_power((float)v * 0.25f, own + w_scale - 254);
                sum[r] += own == 255 || w_scale == 255 ? __uint_as_float(0x7fffffffu) : f;
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int o = 16; o; o >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
            if (lane == r && r < a.rows) {
                float v = sum[r];
                if (a.bias) v += a.bias[n];
                v = activate(v, a.act);
                if (a.residual) v += load_value(a.residual, r * a.ldr + n, a.y_type);
                store_value(a.y, r * a.ldy + n, a.y_type, v);
            }
        }
    }
}

}  // namespace b200
