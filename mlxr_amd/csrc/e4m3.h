// Rounding to 8 bits (e4m3 without infinities, largest value 448): shared by the paged cache and the norms.
#pragma once
#include "qgemm_device.h"

namespace mlxr {

constexpr float kE4m3Top = 448.f;

__device__ __forceinline__ uint32_t e4m3x4(const float* v) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
}
template <int N>
__device__ __forceinline__ float largest(const float (&v)[N]) {
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) top = fmaxf(top, fabsf(v[n]));
  return top;
}

// v / d rounded as division does, for what becomes e4m3: a reciprocal for all of them and two corrections each, the last
// of which is exact (Markstein's theorem: q within an ulp, r the rounded reciprocal, the residue exact).  That holds
// where nothing overflows or comes near the smallest numbers; quotients below 2^-10 become 0 whatever their bits, of v's
// sign.  (4099 tokens of 8 heads of 128 appended to an e4m3 cache: 10.5 us with divisions and every value clamped, 8.3 now,
// 6.1 without scales.)
template <int N>
__device__ __forceinline__ void divide(float (&v)[N], float d) {
  const float r = 1.f / d;
  float q[N];
#pragma unroll
  for (int n = 0; n < N; ++n) q[n] = v[n] * r;
  if (largest(q) < 0x1p80f && fabsf(d) > 0x1p-40f && fabsf(d) < 0x1p40f) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float q1 = __builtin_fmaf(__builtin_fmaf(-q[n], d, v[n]), r, q[n]);
      v[n] = copysignf(__builtin_fmaf(__builtin_fmaf(-q1, d, v[n]), r, q1), q[n]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] /= d;
  }
}

}  // namespace mlxr
