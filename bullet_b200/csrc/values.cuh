// Values of the dense trunk's operators: types of 32, 16 and 8 bits, the 8-bit scales, and activations with their gradients.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "../../include/bullet_b200.h"

namespace b200 {

using bf16 = __nv_bfloat16;
using f16 = __half;
struct e4m3 {
    uint8_t code;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(f16 v) { return __half2float(v); }
__device__ __forceinline__ float to_float(e4m3 v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v.code, __NV_E4M3))); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ f16 from_float<f16>(float v) { return __float2half_rn(v); }

// two neighbours of 16 bits in a word
template <class T>
__device__ __forceinline__ void unpack2(uint32_t w, float& low, float& high);
template <>
__device__ __forceinline__ void unpack2<bf16>(uint32_t w, float& low, float& high) {
    low = __uint_as_float(w << 16), high = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<f16>(uint32_t w, float& low, float& high) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    low = f.x, high = f.y;
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float low, float high);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float low, float high) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<f16>(float low, float high) {
    const __half2 v = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// elements of a type that the launch names
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

__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u; }

// The scale for a largest finite magnitude given by its bits: the smallest power of two from 2^-126 on with magnitude / scale
// <= 448 = 1.75 * 2^8.  1 for a magnitude of 0.
__device__ __forceinline__ uint32_t scale_bits(uint32_t magnitude) {
    if (magnitude == 0) return 127u << 23;
    const int e = (int)(magnitude >> 23) - 8 + ((magnitude & 0x7fffffu) > 0x600000u);
    return (uint32_t)max(e, 1) << 23;
}
__device__ __forceinline__ float one_over_scale(uint32_t scale) { return __uint_as_float((254u << 23) - scale); }

// A sum of products of codes times both scales.  The scales' product may leave fp32's normal numbers where the result does not (or, for
// v = 0, become infinite): then the larger scale first, which takes v out of them only if the result is out as well.
__device__ __forceinline__ bool normal(float v) { return (__float_as_uint(v) & 0x7fffffffu) - 0x800000u < 0x7f000000u; }
__device__ __forceinline__ float scaled(float v, float a, float b) {
    const float s = a * b;
    if (normal(s)) return v * s;
    return fabsf(a) > fabsf(b) ? v * a * b : v * b * a;
}

// The code of v / scale: nearest, halves to even, NaN for what is not finite; what would round up out of fp32 (kTopScale) rounds down.
// For outputs of an activation: what is above 0 stays above 0, what is below 1 stays below 1.
constexpr uint32_t kTopScale = 247u << 23;  // the largest there is: 256 times that is past fp32
static __device__ __noinline__ uint8_t code_of_output(float v, uint32_t scale, int act) {
    uint8_t q = __nv_cvt_float_to_fp8(v * one_over_scale(scale), __NV_SATFINITE, __NV_E4M3);
    if (!finite(v)) return 0x7f;
    if (scale == kTopScale && (q & 0x7f) >= 0x78) q = (q & 0x80) | 0x77;
    if (act == B200_ACT_NONE) return q;
    if (v > 0.f && q == 0) q = 1;
    if (act != B200_ACT_RELU && v > 0.f && v < 1.f && to_float(e4m3{q}) * __uint_as_float(scale) >= 1.f) q--;  // codes above 0 are in the order of their values
    return q;
}

// NaN stays NaN in all of them.
__device__ __forceinline__ float at_least_0(float z) {
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z));
    return z;
}
__device__ __forceinline__ float at_most_1(float z) {
    asm("min.NaN.f32 %0, %0, 0f3F800000;" : "+f"(z));
    return z;
}
__device__ __forceinline__ float activate(float z, int act) {
    if (act == B200_ACT_NONE) return z;
    z = at_least_0(z);
    if (act == B200_ACT_RELU) return z;
    z = at_most_1(z);
    return act == B200_ACT_SCRELU ? z * z : z;
}
template <int N>
__device__ __forceinline__ void activate_all(float (&z)[N], int act) {  // (one question for all)
    if (act == B200_ACT_NONE) return;
    if (act == B200_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < N; k++) z[k] = at_least_0(z[k]);
        return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) z[k] = at_most_1(at_least_0(z[k]));
    if (act == B200_ACT_SCRELU) {
#pragma unroll
        for (int k = 0; k < N; k++) z[k] *= z[k];
    }
}
// dy times the activation's derivative, taken from its output; 0 where that is cut off, whatever dy is.
__device__ __forceinline__ float gradient_from_output(float dy, float y, int act) {
    if (act == B200_ACT_NONE) return dy;
    const bool inside = y > 0.f && (act == B200_ACT_RELU || y < 1.f);
    if (act == B200_ACT_SCRELU) {  // (one instruction, off by 2^-23 at most; the rounded root takes twenty)
        float root;
        asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(y));
        dy *= 2.f * root;
    }
    return inside ? dy : 0.f;
}

}  // namespace b200
