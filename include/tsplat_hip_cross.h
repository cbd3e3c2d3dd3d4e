/*
 * tsplat_hip_cross.h -- C ABI of libtsplat_hip.so's cross attention over a batch of requests: each request's query rows
 * attend to that request's encoder states, both of any length.  It has no counterpart among the reference's libraries;
 * conventions and status codes are those of tsplat_hip.h.
 */
#ifndef TSPLAT_HIP_CROSS_H
#define TSPLAT_HIP_CROSS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Moves with any change to this header's functions or to the plan's layout. */
int tsplat_cross_abi_version(void);

/* The plan of a batch, made on the host and kept while the lengths stay: which workgroup takes which rows and keys.
 * q_lengths, k_lengths [requests] (host): rows and states of each request, in order, either may be 0.  heads a multiple
 * of kv_heads (query head h reads key head h / (heads / kv_heads)), head_dim 1..128; dtype of q, k, v and out: 0 fp32,
 * 1 bf16, 2 fp16; precision of fp32 products: 0 pairs of fp16 values or three bf16 terms of each factor (fp32
 * accuracy: a score to 2^-21 log2 units besides fp32's own error, a weight to 2^-36 of its row's largest, a value of v to
 * 2^-23 of it or 2^-21 of the largest of its feature or of its four neighbours, and none of q, k, v more finely than to
 * 2^-134), 2 two bf16 terms, 1 one (0 for 16-bit types).  Fewer than three terms round finite values to infinities, as
 * bf16 does: one from 3.3962e38 on, two from 3.4027e38 on.
 * Returns the plan's size in ints, or a negative status (-1, -2: sizes; at most 65535 heads, 2^30 - 1 rows times heads of a
 * group, as many states, and 2^32 - 1 threads of a launch).  With plan (host memory of plan_ints ints) it
 * is written there (-3 when too small).  The first TSPLAT_CROSS_HEADER ints describe it. */
#define TSPLAT_CROSS_HEADER 16
int64_t tsplat_cross_plan(const int32_t* q_lengths, const int32_t* k_lengths, int requests, int heads, int kv_heads,
                          int head_dim, int dtype, int precision, int32_t* plan, int64_t plan_ints);
/* Bytes of scratch that calls with this plan need; header: the plan's first ints, on the host. */
int64_t tsplat_cross_scratch_bytes(const int32_t* header);

/* out[t][h] = sum_j softmax_j(scale q[t][h] . k[j][g] + bias[j]) v[j][g], g = h / (heads / kv_heads), over the states j of
 * the request that row t belongs to; zero where it has none, or every bias is -infinity.
 *
 * Sums, maxima and exponents are fp32.  Products of 16-bit types are of the values as they are, summed before scale is
 * multiplied in (those sums must be finite), and of the weights rounded to that type: half a step of each, about as much
 * again as the result's own rounding.
 *
 * q, out: [rows][heads][head_dim], k, v: [states][kv_heads][head_dim] of the plan's type, unit stride within a vector,
 * token and head strides in values (vectors must not overlap, -3); rows and states at least the sums of the plan's lengths; rows past
 * them are not touched.  bias: fp32 [states] or null; a state whose bias is -infinity is not read into any result,
 * whatever it holds; one of +infinity or NaN makes its request's results NaN, and one past 2.3e38 of either sign counts as
 * the type's largest or lowest.  An infinity in q, or in k or v of a state that counts, may come out as a NaN.  scale:
 * positive, and finite times log2 e (-2).
 * header: the plan's first ints (host); plan: all of it on the device, as tsplat_cross_plan wrote it.
 * out must not overlap anything that is read (-3).  scratch: tsplat_cross_scratch_bytes of device memory that no other
 * work uses until the call's kernels are done (-5 when too small, -3 over another argument), 16-byte aligned.  The call
 * only enqueues on `stream` and allocates nothing: it can be captured into a HIP graph as it is. */
int tsplat_cross_attention_async(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                                 int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const float* bias,
                                 float scale, void* out, int64_t out_token, int64_t out_head, const int32_t* header,
                                 const int32_t* plan, void* scratch, int64_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TSPLAT_HIP_CROSS_H */
