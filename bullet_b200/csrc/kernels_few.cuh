// A layer for a few rows: positions that are served one by one or by a handful.
//
// Nothing but W's way from L2 or HBM counts, and the latency around it.  A CTA takes 64 columns of a piece of k, a warp four
// rows of W at a time, sixteen bytes a lane, and eight such loads of a lane are on their way before the first is used; x lies in
// shared memory in fp32.  The CTAs of a cluster share out k: their sums meet in the first one's shared memory and
// are added up in order, so that there is one launch and no workspace.
#pragma once
#include "tensor.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kFewColumns = 64, kFewAhead = 8, kFewStep = 32, kFewChunk = kFewAhead * kFewStep;  // of k: by one load of all threads, by eight
// Up to eight rows: sixteen would not fit in 48 KB of shared memory, and at eight the tiles of kernels_product.cuh come near.  1 / 2 / 4 / 8
// rows here and there, us: 2048 -> 1024 3.6 / 3.9 / 5.4 / 7.9 and 8.4, 512 -> 512 3.2 / 3.6 / 4.2 / 5.2 and 6.8, 512 -> 2048 3.5 / 4.0 / 5.0 /
// 7.0 and 6.9, 2048 -> 16 3.4 / 3.7 / 4.6 / 5.7 and 7.5; in 8 bits 2048 -> 1024 3.8 / 4.3 / 5.5 / 7.4 and 8.2.
constexpr int kFewRowsMost = 8, kFewClusterMost = 8;

struct FewArgs {
    b200_dense_op op;
    int slice;  // of k, of a CTA
};

// Eight elements of a row of W.
template <class T, bool VEC>
struct FewLoad {
    uint32_t w[VEC ? 2 * sizeof(T) : 1];
    T one[VEC ? 1 : 8];
    __device__ __forceinline__ void load(const T* at, int columns) {
        if constexpr (!VEC) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < columns) one[k] = at[k];
        } else if constexpr (sizeof(T) == 2) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
            w[0] = v.x, w[1] = v.y;
        }
    }
    __device__ __forceinline__ void get(float (&v)[8], int columns) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = k < columns ? to_float(one[k]) : 0.f;
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 4; k++) unpack2<T>(w[k], v[2 * k], v[2 * k + 1]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[k / 2] >> 16 * (k & 1)), __NV_E4M3);
                const float2 f = __half22float2(__half2(h));
                v[2 * k] = f.x, v[2 * k + 1] = f.y;
            }
        }
    }
};

template <class T, int ROWS, bool VEC>
static __global__ void __launch_bounds__(256) dense_few_kernel(const FewArgs f) {
    __shared__ float xs[ROWS][kFewChunk];
    __shared__ float sums[8][ROWS][kFewColumns];                // of the warps
    __shared__ float pieces[kFewClusterMost][ROWS][kFewColumns];  // of the cluster's CTAs, in the first one
    const b200_dense_op& a = f.op;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    cluster_arrive();  // (the first CTA has to be there before its memory is written)
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int n0 = (int)(blockIdx.x / ctas) * kFewColumns, n = n0 + 8 * (lane & 7), columns = min(8, a.out - n);
    const int64_t first = (int64_t)rank * f.slice, last = min((int64_t)a.in, first + f.slice);
    const T* w = static_cast<const T*>(a.w) + n;
    float acc[ROWS][8] = {};
    for (int64_t k0 = first; k0 < last; k0 += kFewChunk) {
        FewLoad<T, VEC> ahead[kFewAhead];
        const int64_t k = k0 + 4 * warp + (lane >> 3);
#pragma unroll
        for (int u = 0; u < kFewAhead; u++)
            if (k + u * kFewStep < last && columns > 0) ahead[u].load(w + (k + u * kFewStep) * a.ldw, columns);
        if (k0 > first) __syncthreads();
        for (int i = threadIdx.x; i < ROWS * kFewChunk; i += 256) {
            const int row = i / kFewChunk, c = i % kFewChunk;
            xs[row][c] = row < a.rows && k0 + c < last ? to_float(static_cast<const T*>(a.x)[row * a.ldx + k0 + c]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kFewAhead; u++)
            if (k + u * kFewStep < last && columns > 0) {
                float v[8];
                ahead[u].get(v, columns);
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    const float x = xs[r][u * kFewStep + 4 * warp + (lane >> 3)];
#pragma unroll
                    for (int c = 0; c < 8; c++) acc[r][c] = fmaf(x, v[c], acc[r][c]);
                }
            }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++)
#pragma unroll
        for (int c = 0; c < 8; c++) {
            float v = acc[r][c];
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (lane < 8) sums[warp][r][8 * lane + c] = v;
        }
    __syncthreads();
    cluster_wait();
    for (int i = threadIdx.x; i < ROWS * kFewColumns; i += 256) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) v += (&sums[k][0][0])[i];
        const uint32_t to = of_rank(smem_u32(&pieces[rank][0][0] + i), 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
    }
    cluster_sync();
    if (rank) return;
    for (int i = threadIdx.x; i < ROWS * kFewColumns; i += 256) {
        const int64_t row = i / kFewColumns, column = n0 + i % kFewColumns;
        if (row >= a.rows || column >= a.out) continue;
        float v = 0.f;
        for (uint32_t k = 0; k < ctas; k++) v += (&pieces[k][0][0])[i];
        if constexpr (sizeof(T) == 1) v = scaled(v, a.x_scale[row], a.w_scale[column]);
        if (a.bias) v += a.bias[column];
        v = activate(v, a.act);
        if (a.residual) v += load_value(a.residual, row * a.ldr + column, a.y_type);
        store_value(a.y, row * a.ldy + column, a.y_type, v);
    }
}

}  // namespace b200
