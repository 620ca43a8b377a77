/*
 * mlxr_paged.h -- C ABI of the paged key-value cache: page tables and slot maps built on the
 * device, writes of new keys and values, decode attention over the cache, and tokens moved within it
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

/* Attention of drafted tokens: the last n = starts[r + 1] - starts[r] of row r's lens[r] cached tokens are the nodes of a
 * tree (their keys and values are in the cache, written as any tokens'), queries starts[r] .. starts[r] + n - 1 are theirs.
 * Node i sees the row's tokens before the nodes, and node j where bit j % 64 of mask[token][j / 64] is set, its own
 * included; without a mask nodes 0 .. i (a chain: the next part of a prompt).
 *   q_dev          [tokens, heads, head_dim] of q_dtype (as mlxr_paged_attention), strides in elements, multiples of 16
 *                  bytes; queries from starts[rows] on are padding
 *   starts_dev     [rows + 1] int32, ascending from 0 (mlxr_page_resize gives them); may go past tokens: nodes from there on
 *                  count in n but have no query (what is not listed was not written: masks should not name it)
 *   mask_dev       [tokens, words] of 64 bits, or NULL; nodes from 64 * words on are seen by none
 *   out_dev        [tokens, heads, head_dim] contiguous; padding and nodes that see nothing are zeros
 *   lse_dev        [tokens, heads] fp32 or NULL: as mlxr_paged_attention
 * Tokens of pages outside the cache are left out, and nodes before a row's first token (n > lens[r]).  What a node does not
 * see does not reach it, whatever its bits.  rows up to MLXR_PAGED_MAX_ROWS, rows * kv_heads up to 2^22, tokens * heads
 * up to 2^26 (less, with head_dim above 128); head_dim, strides and the rest as mlxr_paged_attention, without its limits on the distance of pages.  Sums, maxima and the output before
 * its rounding are fp32, whatever the output's type; weights enter their products with the values with 24 bits (bf16 caches) or 22, less
 * what lies below 2^-32 of the largest. */
enum { MLXR_TREE_MAX_WORDS = 64 };
int mlxr_paged_tree_attention_workspace_size(const mlxr_paged_cache* cache, int rows, int tokens, int heads, int table_width,
                                             int q_dtype, int out_dtype, size_t* bytes);
int mlxr_paged_tree_attention(const mlxr_paged_cache* cache, int rows, int tokens, int heads, const void* q_dev, int q_dtype,
                              int64_t q_token_stride, int64_t q_head_stride, const int32_t* table_dev, int64_t table_stride,
                              int table_width, const int32_t* lens_dev, const int32_t* starts_dev, const int64_t* mask_dev,
                              int words, float scale, void* out_dev, int out_dtype, float* lse_dev, void* workspace_dev,
                              size_t workspace_bytes, void* stream);
/* Masks of trees: bit j of mask[token] for each node j of the token's row on its way to the root, itself included.
 *   parents_dev    [tokens] int32: index of a node's parent among its row's nodes, before its own; anything else: a root
 *   positions_dev  [tokens] int32 or NULL: places of the tokens in their rows (mlxr_page_resize's positions; NULL: the
 *                  nodes' indices), from which positions_out gets those in the text, place - index + depth (for rotary
 *                  embeddings; siblings share one)
 *   mask_dev       [tokens, words]; padding sees nothing
 *   positions_out_dev  [tokens] int32 or NULL; -1 for padding */
int mlxr_tree_mask(int rows, int tokens, const int32_t* starts_dev, const int32_t* parents_dev, const int32_t* positions_dev,
                   int words, int64_t* mask_dev, int32_t* positions_out_dev, void* stream);

/* Tokens moved from slots to slots, bit for bit, in `layers` layers whose stores lie k_layer_stride and
 * v_layer_stride elements apart (the cache describes the first; its scales are not used).
 *
 * mlxr_paged_accept keeps the accepted path of each row's drafted tokens: the last n = starts[r + 1] - starts[r] of
 * its lens[r] tokens are the nodes of a tree, at positions c .. c + n - 1, c = lens[r] - n.  Node path[r][j] moves to
 * position c + j, for j < counts[r]; the row then has lens_out[r] = c + the number of nodes kept.
 *   path_dev       [rows, depth] int32, row stride path_stride: ascending.  An entry that is not above the one before it,
 *                  or no node of the row, ends its path
 *   counts_dev     [rows] int32 (negative: 0; past depth: depth)
 *   lens_out_dev   [rows] int32; not lens_dev
 * mlxr_page_resize to lens_out then gives back the pages that the other nodes were in.  Tokens of pages outside the
 * cache are not moved.  No page in two places of the table.  rows up to MLXR_PAGED_MAX_ROWS. */
int mlxr_paged_accept(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride,
                      int rows, const int32_t* table_dev, int64_t table_stride, int table_width, const int32_t* lens_dev,
                      const int32_t* starts_dev, const int32_t* path_dev, int64_t path_stride, int depth,
                      const int32_t* counts_dev, int32_t* lens_out_dev, void* stream);
/* Slots src[i] to slots dst[i]; pairs with a slot outside the cache are left out.  No slot twice in dst, none of dst in
 * src.  Up to 2^27 tokens. */
int mlxr_paged_copy(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride, int tokens,
                    const int32_t* src_dev, const int32_t* dst_dev, void* stream);
/* The new tokens of a mlxr_page_resize (its starts, slots and positions) filled from other rows: those of row r with the
 * tokens at the same positions of row sources[r] (outside [0, rows) or r itself: left out).  Up to 2^27 tokens. */
int mlxr_paged_fork(const mlxr_paged_cache* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride, int rows,
                    const int32_t* table_dev, int64_t table_stride, int table_width, const int32_t* sources_dev,
                    const int32_t* starts_dev, const int32_t* slots_dev, const int32_t* positions_dev, int tokens,
                    void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MLXR_PAGED_H */
