/*
 * mlxr_paged.h -- C ABI of the paged key-value cache: page tables and slot maps built on the
 * device, writes of new keys and values, and decode attention over the cache
 * (libmlxr_qgemm.so; conventions, element types and status codes of mlxr_qgemm.h).
 *
 * A cache holds pages of page_size tokens.  Row r of a batch (a request) owns the pages
 * table[r][0 .. ceil(len/page_size)); token t of it lies in page table[r][t / page_size] at
 * t % page_size, its slot is page * page_size + t % page_size.  Entries past those pages have
 * no meaning.  Keys and values are addressed by strides, so pages may be laid out [head,
 * token, dim] or [token, head, dim], and the stores may be slices of larger tensors; head_dim
 * is contiguous.
 */
#ifndef MLXR_PAGED_H
#define MLXR_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "mlxr_qgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element type beside MLXR_F16 and MLXR_BF16: 8 bits, e4m3 without infinities
 * (largest value 448). */
enum { MLXR_E4M3 = 3 };

/* Rows (requests) of one call of mlxr_page_resize. */
enum { MLXR_PAGED_MAX_ROWS = 4096 };

typedef struct mlxr_paged_cache {
  void* k_dev;
  void* v_dev;
  const float* k_scale_dev; /* [kv_heads] or NULL (1): a stored key element stands for element * scale */
  const float* v_scale_dev;
  int64_t k_stride[3]; /* in elements: page, head, token */
  int64_t v_stride[3];
  int dtype; /* MLXR_F16, MLXR_BF16 or MLXR_E4M3 */
  int num_pages, page_size, kv_heads, head_dim;
} mlxr_paged_cache;

/* Brings the rows from lens[r] tokens to want[r] tokens: pages they no longer need go back to the
 * pool, pages they need more are taken from it, and the slots of the new tokens are listed.
 *   table_dev      [rows, table_width] int32, row stride table_stride; entries of taken pages
 *                  are written, others stay
 *   free_dev       [num_pages] int32, the pool: the first *free_count_dev entries are free pages,
 *                  a stack.  Pages given back are pushed in row order (a row's in the order of
 *                  its tokens), then pages are taken from the top, in row order
 *   lens_out_dev   [rows] int32: want[r], or lens[r] for a row that is refused
 *   free_count_out_dev  [1]
 *   starts_dev     [rows + 1] int32: first new token of each row in the list; the last is their number
 *   slots_dev, positions_dev  [tokens] int32: slot and position of each new token (rows in order,
 *                  a row's tokens in order), -1 past the last; new tokens past `tokens` are not listed
 *   refused_dev    [1]: rows refused, that is left as they were: want[r] is negative or needs more than
 *                  table_width pages, or the pool has too few pages for it and the rows before it that ask for
 *                  any.  So rows that need pages are served as a prefix: after the first that the pool cannot
 *                  serve, every later one that needs a page is refused too, also where pages are left for it
 *                  (rows that need none are not); put those first that should not wait
 * lens_out_dev and free_count_out_dev must not overlap lens_dev and free_count_dev.  lens outside
 * [0, table_width * page_size] are taken as the nearest of these.  num_pages * page_size and
 * rows * table_width * page_size are at most 2^31 - 1.  One launch, no workspace. */
int mlxr_page_resize(int rows, int page_size, int num_pages, int32_t* table_dev, int64_t table_stride, int table_width,
                     const int32_t* lens_dev, const int32_t* want_dev, int32_t* free_dev, const int32_t* free_count_dev,
                     int32_t* lens_out_dev, int32_t* free_count_out_dev, int32_t* starts_dev, int32_t* slots_dev,
                     int32_t* positions_dev, int tokens, int32_t* refused_dev, void* stream);

/* Writes the keys and values of `tokens` tokens into their slots.
 *   k_dev, v_dev   [tokens, kv_heads, head_dim] of x_dtype (MLXR_F32 / MLXR_F16 / MLXR_BF16),
 *                  strides in elements, multiples of 16 bytes as the addresses; head_dim contiguous
 *   slots_dev      [tokens] int32; tokens whose slot lies outside the cache (-1: padding) are
 *                  left out.  No slot twice
 * Elements are divided by their head's scale in fp32 and rounded to nearest even; to e4m3 they
 * saturate at +-448, NaN stays NaN. */
int mlxr_paged_append(const mlxr_paged_cache* cache, int tokens, const void* k_dev, int64_t k_token_stride,
                      int64_t k_head_stride, const void* v_dev, int64_t v_token_stride, int64_t v_head_stride,
                      int x_dtype, const int32_t* slots_dev, void* stream);

/* Attention of one new token per row over its cached tokens (the new one included):
 *   out[r][h] = sum_t softmax_t(scale * q[r][h] . k[t]) v[t],  t in [max(0, len - window), len)
 * (window 0: all), with the keys and values of kv head h / (heads / kv_heads).
 *   q_dev          [rows, heads, head_dim] of q_dtype (MLXR_F16 / MLXR_BF16; the cache's type
 *                  unless that is MLXR_E4M3), strides in elements, multiples of 16 bytes
 *   table_dev      [rows, table_width] int32, row stride table_stride
 *   lens_dev       [rows] int32; a row of length 0 (or less) gives zeros.  Lengths past
 *                  table_width * page_size are taken as that
 *   out_dev        [rows, heads, head_dim] contiguous, at a multiple of 16 bytes, out_dtype MLXR_F32 / MLXR_F16 /
 *                  MLXR_BF16
 *   lse_dev        [rows, heads] fp32 or NULL: natural logarithm of the softmax's sum, -inf for
 *                  an empty row
 * Tokens of pages whose table entry lies outside the cache are left out; a row with no others is an empty
 * row, as one of length 0.  What lies in the cache past a row's tokens is not used, whatever its
 * bits.  head_dim: a multiple of 8 (e4m3: 16), at most 256; keys' and values' strides and addresses
 * are multiples of 16 bytes, the pages and tokens of a store less than 2^31 elements apart;
 * rows * heads is at most 2^24 - 64, the table covers less than 2^31 - 1024 tokens.  Sums,
 * maxima and the output before its rounding are fp32; weights enter their products with the values
 * with 24 bits (bf16 caches) or 22. */
/* Workspace bytes of a call (0: none is needed, workspace_dev may be NULL). */
int mlxr_paged_attention_workspace_size(const mlxr_paged_cache* cache, int rows, int heads, int table_width,
                                        size_t* bytes);
int mlxr_paged_attention(const mlxr_paged_cache* cache, int rows, int heads, const void* q_dev, int q_dtype,
                         int64_t q_row_stride, int64_t q_head_stride, const int32_t* table_dev, int64_t table_stride,
                         int table_width, const int32_t* lens_dev, float scale, int window, void* out_dev, int out_dtype,
                         float* lse_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MLXR_PAGED_H */
