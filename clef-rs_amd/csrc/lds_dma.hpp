// Loads from memory into LDS without registers, as inline assembly: lane l of the
// wave writes 16 bytes at lds_block + 16 l.  The compiler does not see these loads:
// vm_wait_all waits for them, and the wait states that their operands need (M0, and a
// scalar base behind the readfirstlane that makes it) stand in the assembly.
#pragma once
#include "common.hpp"

namespace clef {
namespace {

__device__ __forceinline__ void dma16(const void* src, void* lds_block) {
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_block));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void dma16s(const void* base, uint32_t off, void* lds_block) {
  // the same from a base that is uniform and 32-bit offsets of the lanes
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_block));
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b >> 32)));
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b)));
  const uint64_t sb = (static_cast<uint64_t>(hi) << 32) | lo;
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(sb), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void dma4(const void* src, void* lds_block) {
  // 4 bytes a lane
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_block));
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}
// until at most N of the wave's loads are in flight
template <int N>
__device__ __forceinline__ void vm_wait() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
__device__ __forceinline__ void vm_wait_all() { __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); }

}  // namespace
}  // namespace clef
