// What the entry points of products on the tensor pipe share: maps for TMA, and what a call hears of the one before.
#pragma once
#include <cuda.h>

#include <atomic>

#include "gave_up.h"
#include "op_call.h"

namespace b200 {

constexpr int kSms = 148;  // that products are cut for

// A wait of a kernel before that gave up (Waits) is reported by the next call on its device.
inline int check_gave_up(const char* who, int* word) {
    if (!take_gave_up(word)) return 0;
    return fail(B200_ERR_STATE, "%s: a kernel of a call before on this device waited too long for its own copies or products; that call's outputs are not valid", who);
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline Encode encoder() {
    static std::atomic<void*> found;
    if (!found) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) == cudaSuccess && how == cudaDriverEntryPointSuccess) found = fn;
    }
    return reinterpret_cast<Encode>(found.load());
}
// The result, or its parts, as a stack of matrices, in boxes of 32 rows of 128 (or 64) bytes, swizzled over as many.
inline int make_result_map(CUtensorMap* map, const void* at, int type, int64_t ld, int64_t rows, int64_t cols, int64_t count, int bytes = 128) {
    const Encode encode = encoder();
    if (!encode) return fail(B200_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t row = (cuuint64_t)(rows == 1 ? (cols * type_bytes(type) + 15) / 16 * 16 : ld * type_bytes(type));
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count}, stride[2] = {row, (cuuint64_t)rows * (cuuint64_t)(count > 1 ? ld * type_bytes(type) : row)};
    const cuuint32_t box[3] = {(cuuint32_t)(bytes / type_bytes(type)), 32, 1}, each[3] = {1, 1, 1};
    const CUtensorMapDataType kind = type == B200_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == B200_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult rc = encode(map, kind, 3, const_cast<void*>(at), size, stride, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) on %lld rows of %lld, %lld apart", (int)rc, (long long)rows, (long long)cols, (long long)ld);
    return 0;
}

}  // namespace b200
