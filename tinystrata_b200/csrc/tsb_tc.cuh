// tsb_tc.cuh - the tcgen05 / TMEM helpers that the tensor-core kernels (tsb_mmq.cuh, tsb_cache_prompt.cuh) issue.
#pragma once

#include "tsb_device.cuh"

namespace tsb {

// ------------------------------------------------------------------------------------------------ PTX helpers
// Shared-memory matrix descriptor of a K-major operand tile with the 128-byte swizzle: 8-row groups 1 KB apart.
__device__ __forceinline__ uint64_t pf_sdesc(uint32_t addr) {
    return (uint64_t) ((addr >> 4) & 0x3FFFu) | ((uint64_t) 1 << 16) | ((uint64_t) (1024 >> 4) << 32) |
           ((uint64_t) 1 << 46) | ((uint64_t) 2 << 61);
}
// The mbarrier arrives once every tcgen05.mma this thread issued before it has completed.
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// byte offset of the 16-byte chunk c (values 8c..8c+7) of row r inside a K-major 128-byte-swizzled tile
__device__ __forceinline__ uint32_t sw128(int r, int c) {
    return (uint32_t) ((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}

}  // namespace tsb
