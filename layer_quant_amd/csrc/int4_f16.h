// INT4 nibbles as exact fp16 integers and the fp16 matrix product, shared by the attention kernels
// that work in fp16.
#pragma once

#include "lq_common.h"

namespace lq {
namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mfma_f16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// exact fp16 pair n from the nibbles at bits 3:0 and 19:16 of x: 1032 + n, minus 1032
__device__ __forceinline__ uint32_t nib_pair_f16(uint32_t x) {
  const uint32_t m = ((x ^ 0x00080008u) & 0x000F000Fu) | 0x64006400u;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, m) +
                                          __builtin_bit_cast(f16x2_t, 0xE408E408u));
}

// 8 nibbles of one dword -> fp16 n in slot order of dims (0, 4, 1, 5, 2, 6, 3, 7)
__device__ __forceinline__ u32x4_t decode_octet_f16(uint32_t w) {
  u32x4_t o;
  o.x = nib_pair_f16(w);
  o.y = nib_pair_f16(w >> 4);
  o.z = nib_pair_f16(w >> 8);
  o.w = nib_pair_f16(w >> 12);
  return o;
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}

}  // namespace
}  // namespace lq
