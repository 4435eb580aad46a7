// Loads straight into LDS for kernels that keep a ring of tiles there (tl1_gemm.hip, gemm_i8.hip),
// and the waits and barriers that leave such loads in flight.
#pragma once

#include "common.h"

namespace tz {
namespace {

typedef __attribute__((address_space(3))) void lds_void;
constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw buffer, gfx9 family
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buf(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, kRawBuffer);
}
// 16 bytes per lane from a buffer straight into LDS (no registers): lane l's
// bytes land at dst + 16 l. Offsets past the resource's byte count read zeros.
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t r, void* dst, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, off, 0, 0, 0);
}
// The same load issued from assembly. Around the builtin the compiler cannot tell the
// ring's slots apart and may wait for every outstanding load (vmcnt 0) before each LDS
// read, which stops the ring; here only the waits written out are made. r: the buffer
// resource's four words; lds: the LDS byte address (uniform). The instruction has no
// output registers. M0 needs one wait state before it, and a scalar register that a vector
// instruction has written five: the compiler counts neither inside an asm. The resource's
// words are written by scalar instructions (five wait states before each load make 256 tokens of
// 3840 x 6912 13% slower), and M0, which cannot be declared as written (it is reserved), is used
// for nothing else: the tests of assembly hazards check both in the compiled code.
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u4v buf_words(const void* base, uint32_t bytes) {
    const uint64_t a = (uint64_t)base;
    return u4v{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), (uint32_t)kRawBuffer};
}
__device__ __forceinline__ void to_lds16_asm(u4v r, uint32_t lds, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(off), "s"(r)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// s_barrier without the workgroup fence of __syncthreads(), whose release half
// waits for every outstanding vector memory operation (vmcnt 0), which would
// drain the ring's loads at each chunk. The memory clobber keeps LDS accesses
// on their side of it; LDS-DMA completion is waited for explicitly (wait_vm).
__device__ __forceinline__ void block_barrier() { asm volatile("s_barrier" ::: "memory"); }
// Keeps the memory operations before it ahead of the instructions after it:
// the compiler memory clobber stops IR passes from sinking the loads to their
// first use, the scheduling barrier stops the machine scheduler.
__device__ __forceinline__ void issue_point() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
template <int N> __device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

template <int N> __device__ __forceinline__ void wait_vm_asm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace
}  // namespace tz
