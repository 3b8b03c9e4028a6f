// Products on the tensor pipe: tiles by TMA, descriptors, barriers, tensor memory, for one CTA or a pair (cta_group::1, ::2).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "bulk_copy.cuh"

namespace b200 {

// A wait that gives up: the CTA's other waits then end at once, everybody runs on to the end without issuing more, and the host
// hears of it.  What is waited for are this kernel's own copies and products, which always land; the limit only keeps a broken
// program from hanging the device.  CLUSTER: what is waited for makes ordinary writes of the pair's other CTA visible; else this CTA's, and what TMA
// and the tensor pipe leave (which takes a thread 100 clocks less).
template <bool CLUSTER>
struct WaitsFor {
    volatile int* dead;  // of the CTA, in shared memory
    int* gave_up;        // the host's
    static constexpr uint32_t kAsleepNs = 100000;
    __device__ __forceinline__ static bool arrived(uint64_t* bar, uint32_t parity) {  // by threads of either CTA of a pair
        uint32_t ok;
        // (asleep until then: warps that ask again and again cost power)
        if constexpr (CLUSTER)
            asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
                         : "=r"(ok)
                         : "r"(smem_u32(bar)), "r"(parity), "r"(kAsleepNs)
                         : "memory");
        else
            asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
                         : "=r"(ok)
                         : "r"(smem_u32(bar)), "r"(parity), "r"(kAsleepNs)
                         : "memory");
        return ok != 0;
    }
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
        if (arrived(bar, parity)) return true;
        for (int tries = 0; tries < 20000 && !*dead; tries++)
            if (arrived(bar, parity)) return true;
        if (!*dead) {
            *dead = 1;
            if (gave_up) *reinterpret_cast<volatile int*>(gave_up) = 1;
        }
        return false;
    }
};
using Waits = WaitsFor<true>;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// the same in two halves
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// `local`, an address of shared memory, in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t of_rank(uint32_t local, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
    return at;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// has a map fetched before its first use
__device__ __forceinline__ void know_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// A box of a matrix into shared memory; the bytes are counted at `bar`, a barrier of this CTA or (PAIR) of either.  x in elements,
// a multiple of 16 bytes.
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map),
                     "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
}

// Boxes of a stack of matrices; what lies outside is 0, and not written if the matrix's rows end on 16 bytes.
__device__ __forceinline__ void load_box3(uint32_t to, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to), "l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void store_box3(const CUtensorMap* map, uint32_t from, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(from), "r"(x), "r"(y), "r"(z) : "memory");
}

__device__ __forceinline__ void add_box3(const CUtensorMap* map, uint32_t from, int x, int y, int z) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(from), "r"(x), "r"(y), "r"(z) : "memory");
}

// A tile's descriptor.  Both kinds have rows of 128 bytes with the 128-byte swizzle, eight rows are 1024 bytes.  Along k (K-major):
// a row of the tile per m or n, 128 bytes of k; `column` unused.  Across (MN-major): a row per k, 128 bytes of m or n, the next
// 128 bytes of m or n `column` bytes on.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t smem, uint32_t column) {
    return (uint64_t)((smem & 0x3ffffu) >> 4 | (column >> 4) << 16) | (uint64_t)(64u | 1u << 14 | 2u << 29) << 32;
}
// Form of a product: fp32 sums; type 0 fp16, 1 bf16 (16 bits), or 0 e4m3 (8 bits)
__host__ __device__ constexpr uint32_t product_form(int type, bool a_across, bool b_across, int m, int n) {
    return 1u << 4 | (uint32_t)type << 7 | (uint32_t)type << 10 | (uint32_t)a_across << 15 | (uint32_t)b_across << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
template <bool PAIR, bool BYTES>
__device__ __forceinline__ void multiply(uint32_t sums, uint64_t a, uint64_t b, uint32_t form, bool add) {
#define B200_MULTIPLY(group, kind)                                                                                                      \
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"(sums), \
                 "l"(a), "l"(b), "r"(form), "r"((int)add)                                                                               \
                 : "memory")
    if constexpr (PAIR && BYTES)
        B200_MULTIPLY("2", "f8f6f4");
    else if constexpr (PAIR)
        B200_MULTIPLY("2", "f16");
    else if constexpr (BYTES)
        B200_MULTIPLY("1", "f8f6f4");
    else
        B200_MULTIPLY("1", "f16");
#undef B200_MULTIPLY
}
// arrives at `bar` (of both CTAs of a pair) when the products issued so far are finished
template <bool PAIR>
__device__ __forceinline__ void when_multiplied(uint64_t* bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One whole warp (of each CTA of a pair)
template <bool PAIR>
__device__ __forceinline__ void tensor_memory_take(uint32_t* word, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(word)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(word)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tensor_memory_give(uint32_t at, uint32_t columns) {
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
// 32 columns of a warp's 32 lanes.  (The wait is part of the statement: nothing reads the words before they have arrived.)
__device__ __forceinline__ void load_sums32(uint32_t at, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
        "%26, %27, %28, %29, %30, %31}, [%32];\ntcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(at)
        : "memory");
}
}  // namespace b200
