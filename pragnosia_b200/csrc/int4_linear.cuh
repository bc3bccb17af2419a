// What the kernels of the four-bit linear layer share.
#pragma once
#include "tc_common.cuh"

namespace pgb {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {      // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N_> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N_) : "memory"); }
// Asks for memory to be brought into the L2: 16-byte aligned, a multiple of 16 bytes. It reads nothing that anyone sees, so it may come ahead of the wait for the kernel
// that writes there.
__device__ __forceinline__ void l2_prefetch(const void *p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
// the same for any address and size: the 16-byte pieces that hold any of it
__device__ __forceinline__ void l2_prefetch_around(const void *p, size_t bytes) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15, to = (reinterpret_cast<uintptr_t>(p) + bytes + 15) & ~(uintptr_t)15;
    l2_prefetch(reinterpret_cast<const void *>(from), (uint32_t)(to - from));
}
// the pair of levels in bits 0-3 and 16-19 as bf16 whole numbers less the zero: 0x4300 | q is 128 + q, z2 is 128 + z twice
__device__ __forceinline__ uint32_t level_pair(uint32_t w, uint32_t z2) {
    uint32_t v, d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "n"(0x000f000f), "r"(0x43004300u));       // (w & mask) | magic, one instruction
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(z2));
    return d;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

int int4_tile_launch(const Int4Linear &a, cudaStream_t stream);

}  // namespace pgb
