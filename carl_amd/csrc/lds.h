// lds.h - copies from memory straight into LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace carl {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Past any descriptor's records.
constexpr int kOutside = (int)0xfffffff0u;

// A buffer descriptor of `records` bytes (as an unsigned number) from `base`;
// words that do not lie in them are read as zeros.
__device__ inline i32x4 descriptor(const void* base, int records)
{
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return i32x4{ __builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff),
                  __builtin_amdgcn_readfirstlane(records), 0x00027000 };
}

// 16 bytes a lane from memory to 16 x lane bytes past `lds` (the same for all
// lanes of the wave), without a register.  Written out because the compiler
// would have every later LDS read wait for it; copies are waited for by
// waitCopies(), before the barrier that hands them over.
__device__ inline void copyToLds(i32x4 from, int offset, int more, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(from), "s"(more)
                 : "memory");      // m0 is never live across statements of these kernels
}

__device__ inline void waitCopies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ inline uint32_t ldsAddress(const void* p)
{
    return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p);
}

}  // namespace carl
