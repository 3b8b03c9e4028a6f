// Products of matrices for the dense trunk, and the gradient at a layer's pre-activation.
#pragma once
#include <cuda_runtime.h>

#include "values.cuh"

namespace b200 {

__device__ __forceinline__ float load_value(const void* at, int64_t i, int type) {
    switch (type) {
        case B200_TYPE_F32: return static_cast<const float*>(at)[i];
        case B200_TYPE_BF16: return to_float(static_cast<const bf16*>(at)[i]);
        case B200_TYPE_F16: return to_float(static_cast<const f16*>(at)[i]);
        default: return to_float(static_cast<const e4m3*>(at)[i]);
    }
}
__device__ __forceinline__ void store_value(void* at, int64_t i, int type, float v) {
    switch (type) {
        case B200_TYPE_F32: static_cast<float*>(at)[i] = v; break;
        case B200_TYPE_BF16: static_cast<bf16*>(at)[i] = from_float<bf16>(v); break;
        default: static_cast<f16*>(at)[i] = from_float<f16>(v);
    }
}

// d[m][n] = act(sum over k of a(m, k) b(k, n) + bias[n]) + residual[m][n].  Elements are `along m` / `along k` apart.
struct Product {
    int64_t m, n, k;
    const void *a, *b;
    int64_t a_m, a_k, b_k, b_n;
    int a_type, b_type;
    const float *a_scale_m, *a_scale_k, *b_scale_n;
    const float* bias;
    const void* residual;
    int64_t ldr;
    void* d;
    int64_t ldd;
    int d_type, act;
};

static __global__ void __launch_bounds__(256) product_kernel(Product p) {
    __shared__ float as[16][65], bs[16][65];
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < p.k; k0 += 16) {
        for (int e = threadIdx.x; e < 1024; e += 256) {
            const int i = p.a_k == 1 ? e / 16 : e % 64, j = p.a_k == 1 ? e % 16 : e / 64;
            const int64_t m = m0 + i, k = k0 + j;
            float v = 0.f;
            if (m < p.m && k < p.k) v = load_value(p.a, m * p.a_m + k * p.a_k, p.a_type) * (p.a_scale_k ? p.a_scale_k[k] : 1.f);
            as[j][i] = v;
        }
        for (int e = threadIdx.x; e < 1024; e += 256) {
            const int i = p.b_k == 1 ? e / 16 : e % 64, j = p.b_k == 1 ? e % 16 : e / 64;
            const int64_t n = n0 + i, k = k0 + j;
            bs[j][i] = n < p.n && k < p.k ? load_value(p.b, n * p.b_n + k * p.b_k, p.b_type) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[r][c] = fmaf(as[j][tm * 4 + r], bs[j][tn * 4 + c], acc[r][c]);
        __syncthreads();
    }
    for (int r = 0; r < 4; r++)
        for (int c = 0; c < 4; c++) {
            const int64_t m = m0 + tm * 4 + r, n = n0 + tn * 4 + c;
            if (m >= p.m || n >= p.n) continue;
            float v = acc[r][c];
            if (p.a_scale_m) v *= p.a_scale_m[m] * p.b_scale_n[n];
            v = activate(p.bias ? v + p.bias[n] : v, p.act);
            if (p.residual) v += load_value(p.residual, m * p.ldr + n, p.d_type);
            store_value(p.d, m * p.ldd + n, p.d_type, v);
        }
}

// dz = act'(y) * dy, rounded to dy's type, and the sums of the unrounded values over pieces of the rows: parts[piece][out].
static __global__ void __launch_bounds__(256) dense_dz_kernel(b200_dense_grad_op a, void* dz, float* parts) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.out) return;
    const int64_t first = (int64_t)a.rows * blockIdx.y / gridDim.y, last = (int64_t)a.rows * (blockIdx.y + 1) / gridDim.y;
    float sum = 0.f;
    for (int64_t row = first; row < last; row++) {
        float v = load_value(a.dy, row * a.lddy + c, a.dy_type);
        if (a.act != B200_ACT_NONE) v = gradient_from_output(v, load_value(a.y, row * a.ldy + c, a.y_type) * (a.y_scale ? a.y_scale[row] : 1.f), a.act);
        sum += v;
        if (dz) store_value(dz, row * a.out + c, a.dy_type, v);
    }
    if (parts) parts[(int64_t)blockIdx.y * a.out + c] = sum;
}

}  // namespace b200
