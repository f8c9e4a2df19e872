// dw_tcgen05.cuh -- inline-PTX helpers shared by the tcgen05 (5th-gen tensor core)
// kernels: fences, commits, tensor-memory loads and shared-memory descriptors.
#pragma once

#include <cstdint>

namespace dw {

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 lanes x 16 columns of 32-bit accumulators -> 16 registers per thread.
__device__ __forceinline__ void tc_ld16(uint32_t taddr, int32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor (K-major, swizzled): start address >> 4 in
// bits [0,14); leading-byte offset (unused for swizzled K-major) = 1; the
// constant high word (stride-byte offset = 8 rows * row bytes, version 1,
// swizzle mode) is precomputed on the host.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint64_t hi) {
    return hi | (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16);
}

// Shared-memory matrix descriptor, K-major without swizzle: core matrices of 8
// rows x 16 bytes (rows 16 bytes apart); `lbo` = bytes between the two 16-byte
// halves of a 32-byte K step, `sbo` = bytes between 8-row groups; version 1,
// layout type 0 (no swizzle).
__device__ __forceinline__ uint64_t smem_desc_noswz(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}

// 1 in one lane of a whole warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}

}  // namespace dw
