// Loads from pool rows straight to LDS, and their waits.
#pragma once

#include "ls_common.h"

namespace ls {
namespace {

typedef char __attribute__((address_space(3)))* lds_ptr;

constexpr uint32_t POOL_BYTES = 0x7fffffffu;               // of a page's rows, more than there are

// Sixteen bytes a lane from a resource to LDS at `to` + 16 lane (to: the same in every lane).
// In assembly, since the compiler, where it knows of such a load, waits for all of them before
// the next LDS read of the array; the waits are this file's own (wait_loads).  It writes no
// register.  K and V are read once: the policy of the decode's page loads (against none:
// a decode step of 16 x 16K 76.8 -> 69.5 us, 16 nodes of 16 x 16K 69.6 -> 68.2).
__device__ __forceinline__ void load_to_lds(u4 rsrc, uint32_t off, uint32_t soff, uint32_t to) {
    asm volatile("s_mov_b32 m0, %3\n\t"
                 "s_nop 0\n\t"
                 "buffer_load_dwordx4 %0, %1, %2 offen sc0 nt lds"
                 :: "v"(off), "s"(rsrc), "s"(soff), "s"(to) : "memory", "m0");
}
// Four bytes a lane, which are read again.
__device__ __forceinline__ void load_words_to_lds(u4 rsrc, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\t"
                 "s_nop 0\n\t"
                 "buffer_load_dword %0, %1, 0 offen lds"
                 :: "v"(off), "s"(rsrc), "s"(to) : "memory", "m0");
}
// Until at most N vector memory operations of this wave are outstanding.
template <int N>
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// Of `bytes` from base; what lies outside reads as zeros, without a request.
__device__ __forceinline__ u4 rsrc_of(const char* base, uint32_t bytes) {
    const uint64_t x = (uint64_t)base;
    u4 r;
    r.x = __builtin_amdgcn_readfirstlane((uint32_t)x);
    r.y = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32) & 0xFFFFu);
    r.z = __builtin_amdgcn_readfirstlane(bytes);
    r.w = 0x00020000u;
    return r;
}

}  // namespace
}  // namespace ls
