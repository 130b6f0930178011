// dma.hpp - loads from global memory straight into LDS, written in asm: the compiler, which takes such a load for a pending write of
// all LDS, would wait for every one in flight before each LDS read. They are waited for by count (wait_dma).
#pragma once
#include "common.hpp"

namespace p0 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
// 64 lanes x 16 bytes, buffer resource + lane offset + scalar offset -> LDS at dst + 16 lane
__device__ __forceinline__ void dma16(uint32_t dst, int voff, i32x4 rsrc, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(dst), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}
// 64 lanes x 4 bytes -> LDS at dst + 4 lane
__device__ __forceinline__ void dma4(uint32_t dst, int voff, i32x4 rsrc, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :: "s"(dst), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}
__device__ __forceinline__ i32x4 resource(const void* b) {   // raw, no bounds of its own
  const uint64_t a = (uint64_t)(uintptr_t)b;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)), -1,
               0x00020000};
}
template <int N>
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

}  // namespace p0
