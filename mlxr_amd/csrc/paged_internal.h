// Shared by the paged-cache files (paged_table.hip, paged_attn*).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mlxr_paged.h"
#include "qgemm_device.h"
#include "qgemm_internal.h"

namespace mlxr {

// Host check of a cache's pointers, sizes, strides and alignment; sets the error.
int check_cache(const mlxr_paged_cache* c);

}  // namespace mlxr
