// lds_dma.h -- loads from memory straight into the LDS, and waits for them.
//
// Written as assembly, not with the compiler's builtin: a kernel that keeps several
// stages on their way tells them apart by counting, while the compiler, which
// cannot, would wait for all of them before any LDS read that could meet one.
// They have no output register.  The compiler's own waits come out at most too
// long, since they count fewer loads behind their own than there are.
#pragma once

#include "db_device.h"

namespace dbk {

// A raw buffer resource as four words (see make_rsrc); uniform.
__device__ __forceinline__ u4 dma_rsrc(const void* base, int bytes) {
  const unsigned long long p = reinterpret_cast<unsigned long long>(base);
  return u4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)p),
            (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(p >> 32)),
            (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// Byte address in the LDS of what p points to.
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) char*)p;
}

// 16 bytes a lane: lane l's at `offset` (its own) of the buffer, to lds + 16 l (lds
// uniform); zeros from behind the buffer's end.
__device__ __forceinline__ void dma16(unsigned lds, u4 rsrc, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds),
               "v"(offset), "s"(rsrc)
               : "m0", "memory");
}
// The same for data that is read once: not kept in the caches.
__device__ __forceinline__ void dma16_stream(unsigned lds, u4 rsrc, int offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds),
      "v"(offset), "s"(rsrc)
      : "m0", "memory");
}

// 4 bytes a lane, to lds + 4 l.
__device__ __forceinline__ void dma4(unsigned lds, u4 rsrc, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds),
               "v"(offset), "s"(rsrc)
               : "m0", "memory");
}

// Waits until at most LEFT of the wave's loads are on their way, then for the
// workgroup's other waves.
template <int LEFT>
__device__ __forceinline__ void dma_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void dma_drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Data that no kernel writes while this one runs, read through the scalar cache.
template <class T>
__device__ __forceinline__ T scalar_load(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(unsigned long long)p;
}

}  // namespace dbk
