// 16-bit matrix products and their operands, shared by the prompt kernels.
//
// v_mfma_f32_32x32x16: D[32x32] += A[32x16] B[16x32]. Lane l (col = l mod 32, hi = l / 32) holds A row col
// and B column col with K slots 8 hi .. + 7, and of column col of D the rows 8 (i / 4) + 4 hi + i mod 4,
// i = 0 .. 15.
#pragma once

#include "lds_loads.h"

namespace lq {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t words4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char* lds_t;

template <bool BF>
__device__ __forceinline__ f32x16_t mfma(words4_t a, words4_t b, f32x16_t c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

// Two floats rounded to nearest even, a in the low half.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f16x2_t v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// 16 bytes of LDS.
__device__ __forceinline__ words4_t lds_read16(lds_t at) {
  return *(__attribute__((address_space(3))) words4_t*)at;
}

// A transposing read: each 16 lanes read 4 rows of 16 values, lane j the 8 bytes of row j / 4 and columns
// 4 (j mod 4) .. + 3 (any address), and lane i gets column i's four values. Two of them are an operand of
// eight K slots.
__device__ __forceinline__ words4_t lds_read_columns(lds_t first, lds_t second) {
  typedef __attribute__((address_space(3))) s16x4_t* at_t;
  const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)first));
  const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)second));
  return words4_t{a.x, a.y, b.x, b.y};
}

// A barrier that publishes the waves' LDS reads and writes and leaves their loads from memory in flight
// (__syncthreads waits for those too).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
}

// A descriptor of wave-uniform values in scalar registers, also where the compiler has run out of them.
__device__ __forceinline__ i32x4_t scalar_desc(i32x4_t d) {
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = __builtin_amdgcn_readfirstlane(d[i]);
  return d;
}

// `bytes` of memory for the buffer builtins: what lies past them reads as zero and is not written.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, BUF_DWORD3);
}

// As load_to_lds, for memory that other workgroups read as well.
__device__ __forceinline__ void load_rows_to_lds(i32x4_t desc, lds_t lds, int voff) {
  desc = scalar_desc(desc);
  const uint32_t addr = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(addr), "v"(voff), "s"(desc)
      : "memory", "m0");
}

// The same with 4 bytes per lane.
__device__ __forceinline__ void load_words_to_lds(i32x4_t desc, lds_t lds, int voff) {
  desc = scalar_desc(desc);
  const uint32_t addr = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(addr), "v"(voff), "s"(desc)
      : "memory", "m0");
}

}  // namespace lq
