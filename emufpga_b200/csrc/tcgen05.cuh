// What the kernels on the 5th-generation tensor cores share: descriptors of
// swizzled shared-memory tiles, commits and fences, reads of the accumulator.
#pragma once
#include "device.cuh"

namespace spm {
namespace dev {

// Shared-memory matrix descriptor of a K-major tile in the 128-byte swizzled
// layout: start address >> 4 (bits 0-13), leading byte offset 16 (unused by
// this layout; bits 16-29), stride byte offset 1024 between 8-row groups
// (>> 4 at bit 32), descriptor version 1 (bit 46), swizzle mode 2 = 128-byte
// (bits 61-63).  The start must sit in a 1024-byte aligned swizzle atom; the
// k-th 16-element step inside the 128-byte row adds 32 * k bytes to it.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// Byte offset of 16-byte chunk c (8 bf16 of k = 8c..8c+7) of row r in a
// 128-row tile of the 128-byte swizzled K-major layout: 8-row atoms of 1024
// bytes, chunk index XOR (row mod 8).
__device__ __forceinline__ uint32_t sw128_offset(uint32_t r, uint32_t c) {
    return (r >> 3) * 1024u + (r & 7u) * 128u + ((c ^ (r & 7u)) << 4);
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Sixteen consecutive accumulator columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = __uint_as_float(r[j]);
}

}  // namespace dev
}  // namespace spm
