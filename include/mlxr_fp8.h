/*
 * mlxr_fp8.h -- C ABI of projections in 8-bit floats with a scale for each block of 128 and of what
 * feeds them: RMS norm with the residual's addition, rounding of rows to 8 bits, and the product
 * (libmlxr_qgemm.so; conventions, element types and status codes of mlxr_qgemm.h; 8 bits are
 * MLXR_E4M3 of mlxr_paged.h, largest value 448).
 *
 * Rows in 8 bits: element k of row m stands for q[m][k] * scale[m][k / 128], scales [rows, ceil(K / 128)]
 * fp32.  Weights: w[n][k] stands for w[n][k] * scale[n / 128][k / 128], scales [ceil(N / 128), ceil(K / 128)].
 * The last block of a row or column may be short.
 */
#ifndef MLXR_FP8_H
#define MLXR_FP8_H

#include <stddef.h>
#include <stdint.h>

#include "mlxr_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MLXR_FP8_BLOCK = 128, MLXR_FP8_MAX_SIZE = 1 << 28 };

/* out[m] = s / sqrt(mean(s^2) + eps) * weight,  s = x[m] (+ residual[m]), in fp32, for each of `rows` rows of K.
 *   x_dev         [rows, K] of x_dtype (MLXR_F32 / MLXR_F16 / MLXR_BF16), row stride x_stride elements
 *   residual_dev  the same, row stride residual_stride, or NULL (no addition)
 *   weight_dev    [K] of weight_dtype, or NULL (1)
 *   sum_dev       [rows, K] contiguous of x_dtype: s rounded once (the norm goes by s before that); may be
 *                 residual_dev or x_dev where those are contiguous.  NULL: not wanted
 *   out_dev       [rows, K] contiguous of out_dtype: any float type, or MLXR_E4M3 with
 *   scales_dev    [rows, ceil(K / 128)] fp32 (else NULL): max |out| of a block / 448, 1 for a block of zeros, at least the
 *                 smallest normal float; the 8 bits are out / scale rounded to nearest even.  NaN does not count
 *                 in the maximum and stays NaN; a block with an infinite value is NaN or has an infinite scale.
 *                 out_dev may be x_dev if it has the same type and is contiguous.
 * rows * K up to 2^40, K up to MLXR_FP8_MAX_SIZE. */
int mlxr_rms_norm(int rows, int K, const void* x_dev, int x_dtype, int64_t x_stride, const void* residual_dev,
                  int64_t residual_stride, const void* weight_dev, int weight_dtype, float eps, void* sum_dev, void* out_dev,
                  int out_dtype, float* scales_dev, void* stream);

/* Rows x_dev [rows, K] to 8 bits with scales, as above without the norm. */
int mlxr_quantize_fp8(int rows, int K, const void* x_dev, int x_dtype, int64_t x_stride, void* out_dev, float* scales_dev,
                      void* stream);

/* Weights w_dev [N, K] (contiguous, of w_dtype) to 8 bits with a scale for each 128 x 128. */
int mlxr_quantize_fp8_weight(int N, int K, const void* w_dev, int w_dtype, void* out_dev, float* scales_dev, void* stream);

/* y[m][n] = sum_b x_scale[m][b] * w_scale[n / 128][b] * sum_{k in block b} x[m][k] * w[n][k] (+ bias[n]).
 *   x_dev, w_dev   [M, K], [N, K] e4m3, contiguous, at multiples of 16 bytes; K a multiple of 16
 *   x_scale_dev    [M, ceil(K / 128)], w_scale_dev [ceil(N / 128), ceil(K / 128)] fp32, contiguous
 *   bias_dev       [N] of bias_dtype (MLXR_F32 / MLXR_F16 / MLXR_BF16) or NULL
 *   y_dev          [M, N] contiguous, of y_dtype
 * Sums are fp32 and y is rounded once.  For 16-bit y and more than 16 rows the matrix instruction of 8 bits may be used, which adds
 * eight neighbouring products (k / 8) at a time and drops what each has below 2^-13 of the largest of them; else
 * products and sums within a block are fp32 too (so the last bits of 16-bit y may depend on M).  M and N up to 2^26, K up to 2^22,
 * M * N up to 2^37. */
int mlxr_fp8_matmul_workspace_size(int M, int N, int K, int y_dtype, size_t* bytes); /* 0: none is needed */
int mlxr_fp8_matmul(int M, int N, int K, const void* x_dev, const float* x_scale_dev, const void* w_dev,
                    const float* w_scale_dev, const void* bias_dev, int bias_dtype, void* y_dev, int y_dtype,
                    void* workspace_dev, size_t workspace_bytes, void* stream);
/* The same of rows in 16 or 32 bits: x_dev [M, K] of x_dtype (MLXR_F32 / MLXR_F16 / MLXR_BF16), row stride x_stride elements, is
 * rounded by mlxr_quantize_fp8 into the workspace (at a multiple of 16 bytes, always needed) first. */
int mlxr_fp8_linear_workspace_size(int M, int N, int K, int y_dtype, size_t* bytes);
int mlxr_fp8_linear(int M, int N, int K, const void* x_dev, int x_dtype, int64_t x_stride, const void* w_dev,
                    const float* w_scale_dev, const void* bias_dev, int bias_dtype, void* y_dev, int y_dtype,
                    void* workspace_dev, size_t workspace_bytes, void* stream);
/* Test hook, process-wide: kernel (0: by shape; 1, 2: of few rows; 3 .. 7: tiles, ascending) and splits of K over workgroups of
 * every later mlxr_fp8_matmul and its workspace size. */
int mlxr_fp8_test_force(int kind, int splits);

#ifdef __cplusplus
}
#endif

#endif /* MLXR_FP8_H */
