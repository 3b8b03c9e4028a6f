// What the dense trunk's operator entry points share: the device for the length of a call, and checks of matrices.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bullet_b200.h"
#include "common.h"

#define OP_CK(call)                                                                                       \
    do {                                                                                                  \
        cudaError_t e_ = (call);                                                                          \
        if (e_ != cudaSuccess)                                                                            \
            return b200::fail(B200_ERR_CUDA, "%s failed: %s (%d) at %s:%d", #call, cudaGetErrorString(e_), \
                              (int)e_, __FILE__, __LINE__);                                               \
    } while (0)

namespace b200 {

// Makes `device` current and, at the end, the one that was.
struct OnDevice {
    explicit OnDevice(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device) {
            status = cudaSetDevice(device);
            changed = status == cudaSuccess;
        }
    }
    ~OnDevice() {
        if (changed) cudaSetDevice(before);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    cudaError_t status;
    int before = 0;
    bool changed = false;
};

inline int type_bytes(int type) { return type == B200_TYPE_F32 ? 4 : type == B200_TYPE_E4M3 ? 1 : 2; }
inline bool is_16_bits(int type) { return type == B200_TYPE_BF16 || type == B200_TYPE_F16; }
inline bool is_float(int type) { return type == B200_TYPE_F32 || is_16_bits(type); }
inline bool is_act(int act) { return act >= B200_ACT_NONE && act <= B200_ACT_RELU; }

// A matrix of the caller: there, aligned to its elements, and with rows that do not overlap.
inline int check_matrix(const char* who, const char* what, const void* at, int64_t ld, int64_t rows, int64_t cols, int type) {
    if (!at) return fail(B200_ERR_ARG, "%s: %s is NULL", who, what);
    if ((uintptr_t)at % type_bytes(type)) return fail(B200_ERR_ARG, "%s: %s is not aligned to its elements", who, what);
    if (ld < cols || ld > INT64_MAX / 8 / (rows > 0 ? rows : 1))
        return fail(B200_ERR_ARG, "%s: ld of %s is %lld, with rows of %lld", who, what, (long long)ld, (long long)cols);
    return 0;
}
inline int check_floats(const char* who, const char* what, const void* at) {
    if (!at) return fail(B200_ERR_ARG, "%s: %s is NULL", who, what);
    if ((uintptr_t)at % 4) return fail(B200_ERR_ARG, "%s: %s is not aligned to its elements", who, what);
    return 0;
}
inline int check_workspace(const char* who, const void* at, int64_t bytes, int64_t wanted) {
    if (wanted > 0 && (!at || bytes < wanted || (uintptr_t)at % 16))
        return fail(B200_ERR_ARG, "%s: a 16-byte aligned workspace of %lld bytes is needed", who, (long long)wanted);
    return 0;
}

}  // namespace b200
