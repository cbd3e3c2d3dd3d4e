// Host-side launch of the ragged cross attention; arguments checked by its caller.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cross_plan.h"

namespace tsplat {

struct CrossParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  const float* bias;  // or null
  float scale;
  int heads, kv_heads, group, dim, type, terms, few;
  const CrossItem* items;
  const CrossJoin* joins;
  int item_count, join_count, parts;
  float* partial;
  int32_t* flags;  // of pairs: a workgroup's (item, key head) that they do not serve; null: no pairs
  int vec;  // q, k, v in eights and out in fours are aligned, and dim is a multiple of 8
};
int launch_cross_f32(const CrossParams& p, hipStream_t stream);
int launch_cross_f32_fast(const CrossParams& p, hipStream_t stream);
int launch_cross_pairs(const CrossParams& p, hipStream_t stream);
int launch_cross_16(const CrossParams& p, hipStream_t stream);
// The partial results' join.
int launch_cross_join(const CrossParams& p, hipStream_t stream);

}  // namespace tsplat
