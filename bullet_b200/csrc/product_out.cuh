// What products on the tensor pipe are told, and how whole sums become results: scales, bias, activation, residual, boxes for TMA.
#pragma once
#include "tensor.cuh"
#include "values.cuh"

namespace b200 {

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

}  // namespace b200
