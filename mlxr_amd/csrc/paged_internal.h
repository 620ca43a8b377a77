// Shared by the paged-cache files (paged_table.hip, paged_attn*).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mlxr_paged.h"
#include "qgemm_device.h"
#include "qgemm_internal.h"

namespace mlxr {

// n / d for n < 2^31 by a multiplication: (mulhi(n, mul) + n) >> shift.
struct Divisor {
  uint32_t d = 1, mul = 1, shift = 0;
  Divisor() = default;
  explicit Divisor(int n) : d((uint32_t)n) {
    shift = n > 1 ? 32 - __builtin_clz((uint32_t)n - 1) : 0;
    mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int quotient(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};

// Host check of a cache's pointers, sizes, strides and alignment; sets the error.
int check_cache(const mlxr_paged_cache* c);

}  // namespace mlxr
