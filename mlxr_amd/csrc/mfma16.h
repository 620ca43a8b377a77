// The 16 x 16 x 32 matrix instruction and pairs of 16-bit floats, in bf16 or f16: shared by the paged
// attention and the adapters.
#pragma once
#include "qgemm_device.h"

namespace mlxr {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;

// c[row 4 (l / 16) + i][col l % 16] += sum_k x[row][k] y[col][k] over 32 k; lane l holds k = 8 (l / 16) ..
// + 7 of row (column) l % 16.
template <bool F16>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t x, u32x4_t y, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x), __builtin_bit_cast(f16x8_t, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) return f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
  else return pack_bf16x2(lo, hi);
}
template <bool F16>
__device__ __forceinline__ float unpack(uint32_t w, int h) {
  if constexpr (F16) return f16_bits_to_f32((w >> (16 * h)) & 0xffffu);
  else return __builtin_bit_cast(float, h ? w & 0xffff0000u : w << 16);
}

}  // namespace mlxr
