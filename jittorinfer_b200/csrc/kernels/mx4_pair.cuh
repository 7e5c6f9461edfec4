// Kernels that run as a CTA alone or, PAIR, as pairs of CTAs (consecutive in blockIdx.x) with one tile (cta_group::2): what differs.
#pragma once

#include <atomic>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace mx4 {

using namespace sm100;

// The products so far done: an arrival at the barrier, of a pair at both CTAs' barriers at that place.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t * bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t) 3)
                     : "memory");
    else mma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void alloc_all(uint32_t * slot) {
    if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(slot, 512);
        tmem_relinquish();
    }
}
template <bool PAIR>
__device__ __forceinline__ void free_all(uint32_t at) {
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(512) : "memory");
    else tmem_dealloc(at, 512);
}
// An arrival at a barrier of the pair's first CTA.  What it tells of is in tensor memory (waited for, and fenced by tcgen05.fence) or came through a barrier of its
// own: no other write waits for it.  (As a release for the cluster it took the scale warps 2 thousand cycles a stage.)
template <bool PAIR>
__device__ __forceinline__ void arrive_first(uint64_t * bar) {
    if (PAIR) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(bar)));
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory");
    } else mbar_arrive(bar);
}
__device__ __forceinline__ void both_here() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
// A tile to this CTA's shared memory, told to the barrier of the pair's first CTA.
template <bool PAIR>
__device__ __forceinline__ void load(void * dst, const CUtensorMap * m, uint64_t * bar, int x, int y, int z) {
    if (PAIR) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(bar)));
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(smem_u32(dst)), "l"(m), "r"(at), "r"(x), "r"(y), "r"(z)
            : "memory");
    } else tma_load_3d(dst, m, bar, x, y, z);
}
template <bool PAIR>
__device__ __forceinline__ void load(void * dst, const CUtensorMap * m, uint64_t * bar, int x, int y) {
    if (PAIR) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(bar)));
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(smem_u32(dst)), "l"(m), "r"(at), "r"(x), "r"(y)
            : "memory");
    } else tma_load_2d(dst, m, bar, x, y);
}

// Pairs of CTAs that run at a time (0: not one); known: zeros, of each device.  An answer stands, that there are none too: sizes of buffers go by it.
template <typename... P>
int pair_count(void (*kern)(P...), int threads, int smem, std::atomic<int> (&known)[jib::MAX_DEVICES], std::atomic<unsigned char> (&attr_done)[jib::MAX_DEVICES]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= jib::MAX_DEVICES) return 0;
    int n = known[dev].load();
    if (n == 0) {
        const bool ready = jib::ensure_dyn_smem(kern, smem, attr_done);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (!ready || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
            n = 0;
            (void) cudaGetLastError();           // (else the next launch would be blamed)
        }
        known[dev].store(n > 0 ? n : -1);
    }
    return n > 0 ? n : 0;
}

}  // namespace mx4
