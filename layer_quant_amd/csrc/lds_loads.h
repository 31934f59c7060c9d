// Buffer loads that write LDS directly, and the waits for them, shared by the kernels that keep rings
// of tiles in LDS.
#pragma once

#include "lq_common.h"

namespace lq {

constexpr int BUF_DWORD3 = 0x00020000;  // raw 32-bit buffer, gfx9 family

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

// Raw buffer descriptor (base, stride 0, num_records = bytes, gfx9 dword 3) for wave-uniform
// arguments, so that it lives in 4 SGPRs.
__device__ __forceinline__ i32x4_t make_desc(const void* base, int bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  i32x4_t d;
  d[0] = (int32_t)(uint32_t)a;
  d[1] = (int32_t)((uint32_t)(a >> 32) & 0xffffu);
  d[2] = bytes;
  d[3] = BUF_DWORD3;
  return d;
}

// One 16-byte-per-lane buffer load that writes LDS directly: lane l's 16 bytes (at byte offset
// voff of the buffer; zero past num_records) land at LDS byte address lds + 16 l. Written as
// inline assembly with its own M0 set-up: the compiler's wait insertion for the builtin form did
// not track which LDS buffer each such load targets (it emitted no wait before the reads of one
// buffer and a full wait before the other's), so the waits are explicit (wait_loads) instead.
// M0 is declared clobbered; no other code of this kernel uses M0 (the compiler warns that a
// reserved register in a clobber list is not saved for it).
__device__ __forceinline__ void load_to_lds(i32x4_t desc, const void* lds, int voff) {
  const uint32_t addr =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen nt lds"
      :
      : "s"(addr), "v"(voff), "s"(desc)
      : "memory", "m0");
}

// The same with 4 bytes per lane (lane l's dword lands at lds + 4 l; each dword is range-checked
// on its own).
__device__ __forceinline__ void load_to_lds_b32(i32x4_t desc, const void* lds, int voff) {
  const uint32_t addr =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen nt lds"
      :
      : "s"(addr), "v"(voff), "s"(desc)
      : "memory", "m0");
}

// Wait until at most N vector-memory loads of this wave are outstanding (loads complete in issue
// order, so every load older than the newest N has landed).
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

}  // namespace lq
