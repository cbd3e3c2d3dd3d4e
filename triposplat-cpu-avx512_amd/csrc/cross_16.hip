// Cross attention of bf16 and fp16 values, and the join of partial results.
#include "cross_attention_kernel.h"

namespace tsplat {

int launch_cross_16(const CrossParams& p, hipStream_t stream) {
  return p.type == 1 ? cross::launch_terms<cross::bf16_t, 1>(p, stream)
                     : cross::launch_terms<cross::half_t, 1>(p, stream);
}

namespace {

// Three dependent loads and a launch: 4 to 7 us.
// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p, M the largest m_p.  Four columns of a row a thread; the grid's
// third dimension goes over an item's rows.
constexpr int kJoinThreads = 256, kJoinAhead = 8;
template <class T>
__global__ __launch_bounds__(kJoinThreads) void cross_join_kernel(CrossParams p, int padded, int tile_rows) {
  const CrossJoin join = p.joins[blockIdx.x];
  const int kv = blockIdx.y, columns = padded / 4;
  const int i = blockIdx.z * kJoinThreads + threadIdx.x, row = i / columns, dim = i % columns * 4;
  if (row >= join.rows || dim >= p.dim) return;
  const int64_t part_floats = (int64_t)tile_rows * (padded + 2), next = p.kv_heads * part_floats;
  const float* base = p.partial + ((int64_t)join.first_part * p.kv_heads + kv) * part_floats;
  const float* m = base + tile_rows * padded + row;
  float top = -INFINITY, l = 0.0f;
  floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int n0 = 0; n0 < join.parts; n0 += kJoinAhead) {  // (so many parts' loads are under way at once)
    float mn[kJoinAhead], ln[kJoinAhead];
    floatx4 o[kJoinAhead];
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      const int64_t at = min(n0 + j, join.parts - 1) * next;
      mn[j] = m[at], ln[j] = m[at + tile_rows];
      o[j] = *reinterpret_cast<const floatx4*>(base + at + row * padded + dim);
    }
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      if (n0 + j >= join.parts) break;
      const float new_top = fmaxf(top, mn[j]);
      const float keep = top == new_top ? 1.0f : __builtin_amdgcn_exp2f(top - new_top);
      const float take = mn[j] == new_top ? 1.0f : __builtin_amdgcn_exp2f(mn[j] - new_top);
      l = l * keep + ln[j] * take;
      sum = sum * keep + o[j] * take;
      top = new_top;
    }
  }
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;
  const int at = join.row0 + row;
  T* out = static_cast<T*>(p.out) + (join.token0 + at / p.group) * p.out_token +
           (kv * p.group + at % p.group) * p.out_head + dim;
  T y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = cross::rounded<T>(sum[e] * scale);
  if (p.vec) {
    __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), y, sizeof(y));
  } else {
    for (int e = 0; e < 4; ++e)
      if (dim + e < p.dim) out[e] = y[e];
  }
}

}  // namespace

int launch_cross_join(const CrossParams& p, hipStream_t stream) {
  const int padded = cross_padded_dim(p.dim), rows = cross_tile(padded, p.terms, p.few != 0).wq * 32;
  const dim3 grid(p.join_count, p.kv_heads, (rows * (padded / 4) + kJoinThreads - 1) / kJoinThreads);
  if (p.type == 0)
    cross_join_kernel<float><<<grid, kJoinThreads, 0, stream>>>(p, padded, rows);
  else if (p.type == 1)
    cross_join_kernel<cross::bf16_t><<<grid, kJoinThreads, 0, stream>>>(p, padded, rows);
  else
    cross_join_kernel<cross::half_t><<<grid, kJoinThreads, 0, stream>>>(p, padded, rows);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
