// Copies from memory straight into LDS and the workgroup's meetings about them, for the kernels that keep several buffers in flight
// (qws_fp8.hip, qws_int4.hip).
#pragma once
#include "qws_device.h"

namespace qws {

typedef __attribute__((address_space(3))) void lds_at;
// 1 KB of consecutive bytes of memory into LDS, 16 bytes a lane, past the registers; OFFSET (below 4 KB) moves both places.
// The instruction is written out because the compiler, where it knows of such a copy, waits for all of them before a read of
// LDS; what has arrived is lds_meet's to say.
template <int OFFSET>
__device__ __forceinline__ void lds_copy(const char* from, uint32_t lane_offset, const void* to) {
  const uint32_t at = (uint32_t)(uintptr_t)(lds_at*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"s"(at), "v"(lane_offset), "s"(from), "n"(OFFSET) : "memory", "m0");
}
__device__ __forceinline__ void lds_copy_words(const char* from, uint32_t lane_offset, const void* to) {  // 64 words
  const uint32_t at = (uint32_t)(uintptr_t)(lds_at*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(at), "v"(lane_offset), "s"(from) : "memory", "m0");
}
// Waits until at most N of the wave's newest loads are in flight and its LDS reads are done, then for the workgroup.  One
// statement that no memory access moves across.
template <int N>
__device__ __forceinline__ void lds_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace qws
