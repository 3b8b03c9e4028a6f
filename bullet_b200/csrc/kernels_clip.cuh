// The norm of many tensors together, and what brings it down to a limit.
//
// HBM bound, or L2's where the tensors fit in there; latency for few elements.  The tensors are cut into chunks, which CTAs take in turn.  A thread squares
// 32 elements in fp32 and adds that to a sum in 64 bits, so that long sums lose nothing; where those squares leave fp32's range it squares in 64 bits.  A CTA
// leaves one sum, and who needs the norm adds all of them up in one order: no atomics, equal inputs give equal bits.
#pragma once
#include <cuda_runtime.h>

#include <cstring>

#include "launch.cuh"
#include "values.cuh"

namespace b200 {

constexpr int kClipThreads = 256, kClipMost = 128;  // tensors of a launch
constexpr int kClipCtas = 148 * 8;                  // of a launch, and sums that it leaves
struct ClipBatch {
    const void* g[kClipMost];
    void* out[kClipMost];
    int64_t n[kClipMost];
    int first[kClipMost];  // chunk
    uint8_t type[kClipMost], vec[kClipMost];
    int count, chunks;
};
struct ClipTotal {
    const double* sums;
    int n_sums;
    double max_norm;
    float* norm;
};

constexpr int kClipChunk = kClipThreads * 32;  // elements
// 32 elements of a thread, in pieces of 16 bytes as far apart as the CTA is wide.
template <class T>
struct Piece {
    static constexpr int kEach = 16 / sizeof(T), kMany = 32 / kEach;
    T v[kMany][kEach];
    static __device__ __forceinline__ int64_t at(int64_t chunk, int k) { return chunk * kClipChunk + (k * kClipThreads + (int)threadIdx.x) * kEach; }
    __device__ __forceinline__ void load(const ClipBatch& b, int tensor, int64_t chunk) {
        const T* g = static_cast<const T*>(b.g[tensor]);
        const int64_t n = b.n[tensor];
        const bool vec = b.vec[tensor];
        if (vec && (chunk + 1) * kClipChunk <= n) {
#pragma unroll
            for (int k = 0; k < kMany; k++) {
                const uint4 w = *reinterpret_cast<const uint4*>(g + at(chunk, k));
                memcpy(v[k], &w, 16);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kMany; k++)
#pragma unroll
            for (int i = 0; i < kEach; i++) v[k][i] = at(chunk, k) + i < n ? g[at(chunk, k) + i] : from_float<T>(0.f);
    }
    __device__ __forceinline__ double squares() const {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kMany; k++)
#pragma unroll
            for (int i = 0; i < kEach; i++) sum = fmaf(to_float(v[k][i]), to_float(v[k][i]), sum);
        if (sum > 0x1p-90f && sum < 0x1p120f) return sum;  // (none of them was lost in the sum, or overflowed)
        double exact = 0;
        if (sum == 0.f) {  // (nothing but zeros, as a rule)
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < kMany; k++)
#pragma unroll
                for (int i = 0; i < kEach; i++) any |= __float_as_uint(to_float(v[k][i])) << 1;
            if (!any) return exact;
        }
#pragma unroll
        for (int k = 0; k < kMany; k++)
#pragma unroll
            for (int i = 0; i < kEach; i++) exact = fma((double)to_float(v[k][i]), (double)to_float(v[k][i]), exact);
        return exact;
    }
    // out = share(element)
    template <class F>
    __device__ __forceinline__ void store(const ClipBatch& b, int tensor, int64_t chunk, F share) const {
        T* out = static_cast<T*>(b.out[tensor]);
        const int64_t n = b.n[tensor];
        const bool vec = b.vec[tensor] && (chunk + 1) * kClipChunk <= n;
#pragma unroll
        for (int k = 0; k < kMany; k++) {
            T y[kEach];
#pragma unroll
            for (int i = 0; i < kEach; i++) y[i] = from_float<T>(share(to_float(v[k][i])));
            if (vec) {
                uint4 w;
                memcpy(&w, y, 16);
                __stcs(reinterpret_cast<uint4*>(out + at(chunk, k)), w);
            } else {
#pragma unroll
                for (int i = 0; i < kEach; i++)
                    if (at(chunk, k) + i < n) out[at(chunk, k) + i] = y[i];
            }
        }
    }
};
template <class F>
__device__ __forceinline__ void with_kind(int type, F f) {
    if (type == B200_TYPE_F32)
        f(float{});
    else if (type == B200_TYPE_BF16)
        f(bf16{});
    else
        f(f16{});
}
// The CTA's sum in thread 0, in one order.
__device__ __forceinline__ double cta_sum64(double v, double* shared) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int k = 0; k < kClipThreads / 32; k++) v += shared[k];
    return v;
}

static __global__ void __launch_bounds__(kClipThreads) squares_kernel(const __grid_constant__ ClipBatch b, double* sums) {
    __shared__ double shared[kClipThreads / 32];
    double sum = 0;
    int tensor = 0;
    for (int chunk = blockIdx.x; chunk < b.chunks; chunk += gridDim.x) {
        while (tensor + 1 < b.count && b.first[tensor + 1] <= chunk) tensor++;
        with_kind(b.type[tensor], [&](auto t) {
            Piece<decltype(t)> piece;
            piece.load(b, tensor, chunk - b.first[tensor]);
            sum += piece.squares();
        });
    }
    sum = cta_sum64(sum, shared);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}
// All sums added up: the norm, in every thread.
__device__ __forceinline__ double total_norm(const ClipTotal& t, double* shared) {
    double sum = 0;
    for (int k = threadIdx.x; k < t.n_sums; k += kClipThreads) sum += __ldcg(t.sums + k);
    return sqrt(cta_sum64(sum, shared));
}
static __global__ void __launch_bounds__(kClipThreads) norm_kernel(const ClipTotal t) {
    __shared__ double shared[kClipThreads / 32];
    step_begin(nullptr);
    const double norm = total_norm(t, shared);
    if (threadIdx.x == 0) *t.norm = (float)norm;
}
// out = share * g, chunks from the last one back: those are still in L2.
static __global__ void __launch_bounds__(kClipThreads) clip_kernel(const __grid_constant__ ClipBatch b, const ClipTotal t) {
    __shared__ double shared[kClipThreads / 32];
    step_begin(nullptr);
    const double norm = total_norm(t, shared);
    if (threadIdx.x == 0 && blockIdx.x == 0 && t.norm) *t.norm = (float)norm;
    const bool clips = norm > t.max_norm && norm < 0x1p1023;
    const double ratio = clips ? t.max_norm / norm : 1.0;
    const bool tiny = ratio < 0x1p-100;  // (below fp32's normal numbers a share would lose bits, or all: it stays in 64 then)
    const float share = (float)ratio;
    int tensor = b.count - 1;
    for (int chunk = b.chunks - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        while (b.first[tensor] > chunk) tensor--;
        if (!b.out[tensor] || (!clips && b.g[tensor] == b.out[tensor])) continue;
        with_kind(b.type[tensor], [&](auto k) {
            Piece<decltype(k)> piece;
            piece.load(b, tensor, chunk - b.first[tensor]);
            if (__builtin_expect(tiny, 0))
                piece.store(b, tensor, chunk - b.first[tensor], [=](float x) { return (float)(x * ratio); });
            else
                piece.store(b, tensor, chunk - b.first[tensor], [=](float x) { return x * share; });
        });
    }
}

}  // namespace b200
