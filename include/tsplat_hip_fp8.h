/*
 * tsplat_hip_fp8.h -- C ABI of libtsplat_hip.so's 8-bit rows and products: values in e4m3 with a power-of-two scale
 * for each block of 128 of a row, and a Linear on such rows and weights with the step that follows it.  They have no
 * counterpart among the reference's libraries; conventions and status codes are those of tsplat_hip.h: every array
 * is a device pointer of the current device, extents are checked before any launch (-6), the calls only enqueue on
 * `stream` (hipStream_t) and allocate nothing, so they can be captured into a HIP graph as they are.
 */
#ifndef TSPLAT_HIP_FP8_H
#define TSPLAT_HIP_FP8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Moves with any change to this header's functions. */
int tsplat_fp8_abi_version(void);

/* Rows of K values in 8 bits.  codes: [rows][Kp], Kp = K rounded up to 128, e4m3 (1 sign, 4 exponent, 3 fraction bits,
 * largest 448, no infinity), zero past K; exponents: [rows][Ke], Ke = Kp / 128 rounded up to 4, block b of a row
 * stands for codes * 2^(exponents[b] - 127); 127 past the last block.  codes 16-byte aligned, exponents 4-byte (-4): a
 * run of rows is such rows again.
 *
 * The scale is the smallest power of two, 2^-127 at least, that brings the block's largest finite magnitude to 448 or
 * below (1 for a block without one), a code the nearest value of x / scale, ties to even; an infinity or NaN gives a
 * NaN.  (An fp32 value of 248 * 2^120 and more rounds to 2^128, which is an infinity to fp32.)
 * dtype of x: 0 fp32, 1 bf16, 2 fp16; rows x_stride values apart.  rows up to 2^27, K up to 2^20 (-2).  codes and
 * exponents must not overlap each other or x (-3). */
int tsplat_fp8_quantize_async(const void* x, int dtype, int64_t x_stride, int rows, int K, uint8_t* codes,
                              uint8_t* exponents, void* stream);

/* y[m][n] = sum_k x8[m][k] w8[n][k] + bias[n];  y = gelu_tanh(y) with activation 1 (0: none);
 * out[m][n] = y * gate[m / rows_per_batch][n] + residual[m][n].
 *
 * x8: the 8-bit rows of x (dtype, x_stride as above), made within the call, or with x null the rows at x_codes,
 * x_exponents; w8: N rows of K as above.  Sums are held in fp32.  Products:
 *   out_dtype 0, or at most 64 rows: exact (a value below 2^-126 is first rounded to a multiple of 2^-133);
 *   out_dtype 1 and 2 beyond 64 rows: those of each 8 neighbouring values are brought to the largest one's exponent and
 *   cut at 2^-13 of its power of two: 2^-10 of the magnitudes that are summed at most, 1.5e-5 of a sum of random signs or
 *   so.  Where the terms cancel that is more of the sum, and the same row may differ by it between a call of 64 rows and
 *   one of more.
 * bias [N], gate (rows gate_stride floats apart, 0 for one row that serves all) and residual may be null; residual and
 * out are of out_dtype, rows residual_stride and out_stride values apart; out may be residual itself (same pointer and
 * stride) and must not overlap anything else that is read (-3).
 * scratch: at least tsplat_fp8_linear_scratch_bytes(M, K, N, x != null) of device memory that no other work uses until
 * the call's kernels are done (-5 when too small, -3 over another argument), 16-byte aligned.  The size is 0 for a
 * call that needs none, and for sizes that the call refuses. */
int64_t tsplat_fp8_linear_scratch_bytes(int M, int K, int N, int x_given);
int tsplat_fp8_linear_async(const void* x, int x_dtype, int64_t x_stride, const uint8_t* x_codes,
                            const uint8_t* x_exponents, const uint8_t* w_codes, const uint8_t* w_exponents,
                            const float* bias, int activation, const float* gate, int64_t gate_stride,
                            int64_t rows_per_batch, const void* residual, int64_t residual_stride, void* out,
                            int out_dtype, int64_t out_stride, int M, int K, int N, void* scratch,
                            int64_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TSPLAT_HIP_FP8_H */
