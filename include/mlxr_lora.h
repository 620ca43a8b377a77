/*
 * mlxr_lora.h -- C ABI of the low-rank adapters of many requests beside shared projections
 * (libmlxr_qgemm.so; conventions, element types and status codes of mlxr_qgemm.h).
 *
 *   out[t] = y[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T,   a = ids[t]
 *
 * for each of `count` projections that read the same x (q/k/v, gate/up); y is the shared
 * projection's output (mlxr_qgemm_run and its kin).  Tokens of any adapters may follow each
 * other in any order; a token without one (ids[t] outside [0, adapters)) keeps y[t].  An output may
 * be its y and must not overlap anything else that the call reads.
 */
#ifndef MLXR_LORA_H
#define MLXR_LORA_H

#include <stddef.h>
#include <stdint.h>

#include "mlxr_qgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MLXR_LORA_MAX_ADAPTERS = 4096, MLXR_LORA_MAX_RANK = 128, MLXR_LORA_MAX_TOKENS = 1 << 20, MLXR_LORA_MAX_SIZE = 1 << 28 };

typedef struct mlxr_lora_item {
  const void* a_dev; /* [adapters, rank, K] of x's type, contiguous */
  const void* b_dev; /* [adapters, N, rank] of x's type, contiguous */
  const void* y_dev; /* [tokens, N] contiguous */
  void* out_dev;     /* [tokens, N] contiguous; may be y_dev */
  int N, y_dtype;    /* of y and out: MLXR_F32 / MLXR_F16 / MLXR_BF16 */
} mlxr_lora_item;

/* Workspace bytes of mlxr_lora_apply (0: none is needed, workspace_dev may be NULL).  Only the items' N are read. */
int mlxr_lora_workspace_size(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank,
                             size_t* bytes);

/* x_dev [tokens, K] of x_dtype (MLXR_F16 / MLXR_BF16), row stride x_stride elements; K and x_stride
 * multiples of 8, K and N up to MLXR_LORA_MAX_SIZE, rank a multiple of 8 up to MLXR_LORA_MAX_RANK; x, A and B at multiples of 16 bytes.
 *   ids_dev     [tokens] int32
 *   scales_dev  [adapters] fp32 or NULL (1)
 *   ranks_dev   [adapters] int32 or NULL (rank): rank of each adapter, up to `rank`; what A and B hold
 *               past an adapter's rank is not used, whatever its bits
 * Sums are fp32, out is rounded once.  x . A^T enters the second product with all its bits (bf16), or to 2^-20 of each of its
 * elements (f16). */
int mlxr_lora_apply(int count, const mlxr_lora_item* items, int tokens, int K, int adapters, int rank, const void* x_dev,
                    int x_dtype, int64_t x_stride, const int32_t* ids_dev, const float* scales_dev,
                    const int32_t* ranks_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MLXR_LORA_H */
