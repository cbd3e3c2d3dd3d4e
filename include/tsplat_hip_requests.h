/*
 * tsplat_hip_requests.h -- C ABI of the operators of libtsplat_hip.so that serve a batch of several requests:
 * low-rank adapters beside a shared Linear, a branch's norm, gate and residual with the next norm, and rotary
 * positions of several axes.  They have no counterpart among the reference's libraries; conventions and status
 * codes are those of tsplat_hip.h: every array is a device pointer of the current device, extents are checked
 * before any launch (-6), the calls only enqueue on `stream` (hipStream_t) and allocate nothing, so they can be
 * captured into a HIP graph as they are.
 */
#ifndef TSPLAT_HIP_REQUESTS_H
#define TSPLAT_HIP_REQUESTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Moves with any change to this header's functions. */
int tsplat_requests_abi_version(void);

/* ---------------- low-rank adapters ------------------------------------- */

/* out[m][n] = y[m][n] + scale[a] * sum_r (sum_k x[m][k] down[a][r][k]) up[a][n][r],  a = rows[m];
 * out[m] = y[m] where rows[m] is not in [0, slots) or rank[a] <= 0 (nothing is written there when out is y).
 *
 * y, x, out: fp32, M rows of N, K, N values, y_stride / x_stride / out_stride floats apart.  out may be y itself
 * (same pointer and stride); it must not overlap y otherwise, nor anything else that is read (-3).
 * dtype of the adapters: 0 fp32, 1 bf16, 2 fp16.  Their values are laid out in tiles that one wave reads as one
 * piece, zero past K, N and each adapter's rank:
 *   down: [slots][ceil(R/16)][ceil(K/32)][4][16][8], value (r, k) at [r/16][k/32][k%32/8][r%16][k%8];
 *   up:   [slots][ceil(N/16)][ceil(R/32)][4][16][8], value (n, r) at [n/16][r/32][r%32/8][n%16][r%8];
 * fp32: [slots][..][..][3][4][16][8] bf16, three planes whose sum is the value: its upper 16 bits, those of what is
 * left, and those of what is left then.  R = max_rank, 1..512; rank[a] <= R (a larger one counts as R).  16-byte
 * aligned (-4).  M up to 2^27, K and N up to 2^20, slots up to 2^20 (-2).  A row of x that holds an infinity or NaN
 * gives NaN.  A product of two factors is off by less than 2^-21 of it with fp32 adapters, 2^-22 with fp16, besides
 * its sum's roundings.  The factors (x, the adapter, the inner sums) count in steps of 2^-133 where fp32's own are
 * finer, below 2^-110.
 * scratch: at least tsplat_low_rank_scratch_bytes(...) of device memory that no other work uses until the call's
 * kernels are done (-5 when too small, -3 over another argument), 16-byte aligned.
 * The size is 0 for a call that needs none, and for sizes or a dtype that the call refuses. */
int64_t tsplat_low_rank_scratch_bytes(int M, int K, int N, int slots, int max_rank, int dtype);
int tsplat_low_rank_add_async(const float* y, int64_t y_stride, const float* x, int64_t x_stride,
                              const int32_t* rows, const void* down, const void* up, const float* scale,
                              const int32_t* rank, float* out, int64_t out_stride, int M, int K, int N,
                              int slots, int max_rank, int dtype, void* scratch, int64_t scratch_bytes,
                              void* stream);

/* ---------------- norm, gate, residual, norm ---------------------------- */

/* h' = post(h);  x' = residual_scale * x + gate[b] * h';  out = x';  normed = pre(x') * (1 + scale[b]) + shift[b],
 * over `rows` (below 2^31) rows of `cols` fp32 values; b = row / rows_per_batch.
 * norm kinds: 0 none (post only), 1 LayerNorm, 2 RMS norm (x / sqrt(mean(x^2) + eps)); each with its weight and
 * bias [cols], either null.  gate null: 1; scale and shift: both or neither; their rows mod_stride floats apart
 * (gate: gate_stride), 0 for one row that serves every b.  x, h, out, normed rows are x_stride ... floats apart.
 * Statistics are sums in fp32: a row whose squares pass its range has no norm.  out may be x, normed may be h (same
 * pointer and stride); other overlaps are refused (-3). */
int tsplat_residual_norm_async(const float* x, int64_t x_stride, const float* h, int64_t h_stride, float* out,
                               int64_t out_stride, float* normed, int64_t normed_stride, int64_t rows, int cols,
                               float residual_scale, const float* gate, int64_t gate_stride, int post_kind,
                               const float* post_weight, const float* post_bias, float post_eps, int pre_kind,
                               const float* pre_weight, const float* pre_bias, float pre_eps, const float* scale,
                               const float* shift, int64_t mod_stride, int64_t rows_per_batch, void* stream);

/* ---------------- rotary positions of several axes ---------------------- */

/* Vectors (b, l, h) of `parts` (1..3) tensors, part i read at x + i * part_stride + b * batch_stride +
 * l * token_stride + h * head_stride (floats; unit stride within the vector) and written to out_i as [B, H, L, D]
 * (out_bhld) or [B, L, H, D], contiguous.  Parts 0 and 1 (q and k) are turned: pair p of D/2 by
 * positions[..][axis[p]] * turns[p] revolutions (turns: double, the angle's frequency / 2 pi), and, with a gamma
 * [H, D], become y * sqrt(D) / max(||y||, eps) * gamma.  Part 2 (v) is copied.  A pair is (2p, 2p + 1) with
 * interleaved, else (p, p + D/2).
 * positions: [position_batches][L][axes], position_batches 1 or B, int32 (position_type 0) or fp32 (1); an axis[p]
 * outside [0, axes) counts as 0.  axes 1..8; D even, 2..512; H up to 2^16, B * L below 2^31.  The outputs must not
 * overlap each other, the memory that x spans or anything else that is read (-3). */
int tsplat_rope_axes_async(const float* x, int64_t part_stride, int64_t batch_stride, int64_t token_stride,
                           int64_t head_stride, int parts, const float* gamma0, const float* gamma1,
                           float* out0, float* out1, float* out2, const void* positions, int position_type,
                           int position_batches, int axes, const double* turns, const int32_t* axis,
                           int interleaved, float eps, int B, int L, int H, int D, int out_bhld, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TSPLAT_HIP_REQUESTS_H */
