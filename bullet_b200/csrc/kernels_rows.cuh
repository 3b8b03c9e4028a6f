// Kernels over the rows of a matrix: root-mean-square norm and its gradient, 8-bit packing.
#pragma once
#include <cuda_runtime.h>

#include "values.cuh"

namespace b200 {

constexpr int kRowThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* shared) {  // the same bits in every thread; `shared`: one float per warp
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int k = 0; k < (int)blockDim.x / 32; k++) v += shared[k];
    __syncthreads();
    return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int k = 0; k < (int)blockDim.x / 32; k++) v = max(v, shared[k]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ uint32_t finite_magnitude(float v) { return finite(v) ? __float_as_uint(v) & 0x7fffffffu : 0u; }

// A CTA per row at a time, elements one by one.
template <class TX, class TY>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_kernel(b200_rms_norm_op a) {
    __shared__ float sums[kRowThreads / 32];
    __shared__ uint32_t largest[kRowThreads / 32];
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
        const float rstd = 1.f / sqrtf(block_sum(v, sums) / (float)a.cols + a.eps);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
        auto normed = [&](int c) { return total(c) * rstd * (a.weight ? a.weight[c] : 1.f); };
        if constexpr (sizeof(TY) == 1) {
            uint32_t m = 0;
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) m = max(m, finite_magnitude(normed(c)));
            const uint32_t scale = scale_bits(block_max(m, largest));
            if (threadIdx.x == 0) a.scale[row] = __uint_as_float(scale);
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) static_cast<uint8_t*>(a.y)[row * a.ldy + c] = code_of(normed(c), one_over_scale(scale));
        } else {
            for (int c = threadIdx.x; c < a.cols; c += kRowThreads) static_cast<TY*>(a.y)[row * a.ldy + c] = from_float<TY>(normed(c));
        }
    }
}

template <class TX, class TD>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_dx_kernel(b200_rms_norm_grad_op a) {
    __shared__ float sums[kRowThreads / 32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* s = static_cast<const TX*>(a.sum) + row * a.lds;
        const TD* dy = static_cast<const TD*>(a.dy) + row * a.lddy;
        const TX* ds = a.dsum ? static_cast<const TX*>(a.dsum) + row * a.ldds : nullptr;
        const float rstd = a.rstd[row];
        auto g = [&](int c) { return to_float(dy[c]) * (a.weight ? a.weight[c] : 1.f); };
        float v = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) v = fmaf(g(c), to_float(s[c]) * rstd, v);
        const float mean = block_sum(v, sums) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) {
            const float dx = rstd * (g(c) - to_float(s[c]) * rstd * mean);
            static_cast<TX*>(a.dx)[row * a.lddx + c] = from_float<TX>(ds ? dx + to_float(ds[c]) : dx);
        }
    }
}

// Sums over a piece of the rows, a thread per column: parts[piece][cols].
template <class TX, class TD>
static __global__ void __launch_bounds__(kRowThreads) rms_norm_dweight_kernel(b200_rms_norm_grad_op a, float* parts) {
    const int c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    float v = 0.f;
    for (int64_t row = first; row < last; row++)
        v = fmaf(to_float(static_cast<const TD*>(a.dy)[row * a.lddy + c]), to_float(static_cast<const TX*>(a.sum)[row * a.lds + c]) * a.rstd[row], v);
    parts[(int64_t)blockIdx.y * a.cols + c] = v;
}
static __global__ void __launch_bounds__(kRowThreads) add_parts_kernel(const float* parts, int n_parts, int cols, float* out) {
    const int c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= cols) return;
    float v = 0.f;
    for (int k = 0; k < n_parts; k++) v += parts[(int64_t)k * cols + c];
    out[c] = v;
}

template <class TX>
static __global__ void __launch_bounds__(kRowThreads) pack8_rows_kernel(b200_pack8_op a) {
    __shared__ uint32_t largest[kRowThreads / 32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
        uint32_t m = 0;
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads) m = max(m, finite_magnitude(to_float(x[c])));
        const uint32_t scale = scale_bits(block_max(m, largest));
        if (threadIdx.x == 0) a.scale[row] = __uint_as_float(scale);
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads)
            static_cast<uint8_t*>(a.q)[row * a.ldq + c] = code_of_output(to_float(x[c]), one_over_scale(scale), __uint_as_float(scale), a.act);
    }
}

// By column: a thread per column and piece of the rows.  Scales are in the order of their bits and none is 0, so the largest of
// the pieces' is the column's; a column without a finite value but 0 is left at 0, which pack8_columns_kernel takes for 1 and
// whose first piece writes 1 there: the others take either as 1.
template <class TX>
static __global__ void __launch_bounds__(kRowThreads) column_scales_kernel(b200_pack8_op a) {
    const int c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    uint32_t m = 0;
    for (int64_t row = first; row < last; row++) m = max(m, finite_magnitude(to_float(static_cast<const TX*>(a.x)[row * a.ldx + c])));
    if (m) atomicMax(reinterpret_cast<uint32_t*>(a.scale) + c, scale_bits(m));
}
template <class TX>
static __global__ void __launch_bounds__(kRowThreads) pack8_columns_kernel(b200_pack8_op a) {
    const int c = blockIdx.x * kRowThreads + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    volatile uint32_t* at = reinterpret_cast<uint32_t*>(a.scale) + c;
    uint32_t scale = *at;
    if (scale == 0) {
        scale = scale_bits(0);
        if (blockIdx.y == 0) *at = scale;
    }
    for (int64_t row = first; row < last; row++)
        static_cast<uint8_t*>(a.q)[row * a.ldq + c] =
            code_of_output(to_float(static_cast<const TX*>(a.x)[row * a.ldx + c]), one_over_scale(scale), __uint_as_float(scale), a.act);
}

template <class TY>
static __global__ void __launch_bounds__(kRowThreads) unpack8_kernel(b200_unpack8_op a) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x)
        for (int c = threadIdx.x; c < a.cols; c += kRowThreads)
            static_cast<TY*>(a.y)[row * a.ldy + c] =
                from_float<TY>(to_float(static_cast<const e4m3*>(a.q)[row * a.ldq + c]) * a.scale[a.by_column ? c : row]);
}

}  // namespace b200
