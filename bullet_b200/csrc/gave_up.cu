// Words of waits that gave up, one per device, and b200_op_dense_gave_up.
//
// They are memory of the library image that both sides may touch at any time; kernels touch them only if there is something to report.
// (In a source without kernels: a module with such a variable is loaded as a whole when CUDA starts, also where networks alone are
// trained.  With all product kernels in it a process took the same 755 MB for its first network, and 0.8 to 1.9 s either way.)
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/bullet_b200.h"
#include "common.h"
#include "gave_up.h"

namespace b200 {

constexpr int kDevices = 64, kStride = 16;  // (a cache line each)
static __managed__ int g_gave_up[kDevices * kStride];

int* gave_up_word(int device) {
    static std::atomic<signed char> known[kDevices];  // 0 not asked yet, 1 yes, -1 no
    if (device < 0 || device >= kDevices) return nullptr;
    if (known[device] == 0) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // (the first call may be one that a stream captures)
        cudaThreadExchangeStreamCaptureMode(&mode);
        int concurrent = 0;
        if (cudaDeviceGetAttribute(&concurrent, cudaDevAttrConcurrentManagedAccess, device) != cudaSuccess) concurrent = 0;
        if (concurrent) {  // (hints: the words stay in host memory)
            cudaMemAdvise(g_gave_up, sizeof g_gave_up, cudaMemAdviseSetPreferredLocation, cudaCpuDeviceId);
            cudaMemAdvise(g_gave_up, sizeof g_gave_up, cudaMemAdviseSetAccessedBy, device);
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
        cudaGetLastError();
        known[device] = concurrent ? 1 : -1;
    }
    return known[device] > 0 ? g_gave_up + kStride * device : nullptr;
}

bool take_gave_up(int* word) { return word && __atomic_load_n(word, __ATOMIC_RELAXED) && __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL); }

}  // namespace b200

extern "C" int b200_op_dense_gave_up(int device, int32_t** word) {
    if (!word) return b200::fail(B200_ERR_ARG, "op_dense_gave_up: null result");
    *word = b200::gave_up_word(device);
    return 0;
}
