// Products of the 5th-generation tensor cores issued from a warp that stays whole: every lane runs the loop and one of them issues, so that addresses
// and descriptors are values of the warp.  With a branch for a single lane around the loop each instruction took about 130 cycles
// to issue, twice what a 128 x 128 x 16 product takes; this way the products run back to back.
#pragma once

#include "tc_common.cuh"

namespace lumen {
namespace tc {

__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// d (+)= a . b^T, both operands in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, bool accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// The first operand in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, bool accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// One arrival at `bar` when the products issued so far are complete.
__device__ __forceinline__ void commit_one(uint64_t *bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(saddr(bar)) : "memory");
}
// wait_or_failed by all lanes; the answer is the warp's.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *failed, DeviceStatus *status, int site) {
    return __all_sync(0xffffffffu, wait_or_failed(bar, parity, failed, status, site));
}

}  // namespace tc
}  // namespace lumen
