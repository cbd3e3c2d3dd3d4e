// Cross attention of bf16 and fp16 values, and the join of partial results.
#include "cross_attention_kernel.h"

namespace tsplat {

int launch_cross_16(const CrossParams& p, hipStream_t stream) {
  return p.type == 1 ? cross::launch_terms<cross::bf16_t, 1>(p, stream)
                     : cross::launch_terms<cross::half_t, 1>(p, stream);
}

namespace {

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p, M the largest m_p; a workgroup joins one item's rows of one head.
// Four columns a thread.
template <class T>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossParams p, int padded, int tile_rows) {
  const CrossJoin join = p.joins[blockIdx.x];
  const int kv = blockIdx.y, columns = padded / 4;
  const int64_t part_floats = (int64_t)tile_rows * (padded + 2);
  const float* base = p.partial + ((int64_t)join.first_part * p.kv_heads + kv) * part_floats;
  const int64_t next = p.kv_heads * part_floats;
  for (int i = threadIdx.x; i < join.rows * columns; i += 256) {
    const int row = i / columns, dim = i % columns * 4;
    if (dim >= p.dim) continue;
    const float* m = base + tile_rows * padded + row;
    float top = -INFINITY;
    for (int n = 0; n < join.parts; ++n) top = fmaxf(top, m[n * next]);
    floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (int n = 0; n < join.parts; ++n) {
      const float mn = m[n * next];
      const float w = mn == top ? 1.0f : __builtin_amdgcn_exp2f(mn - top);
      l += w * m[n * next + tile_rows];
      sum += w * *reinterpret_cast<const floatx4*>(base + n * next + row * padded + dim);
    }
    const float scale = l == 0.0f ? 0.0f : 1.0f / l;
    const int at = join.row0 + row;
    T* out = static_cast<T*>(p.out) + (join.token0 + at / p.group) * p.out_token +
             (kv * p.group + at % p.group) * p.out_head + dim;
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(sum[e] * scale);
    if (p.vec) {
      __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), y, sizeof(y));
    } else {
      for (int e = 0; e < 4; ++e)
        if (dim + e < p.dim) out[e] = y[e];
    }
  }
}

}  // namespace

int launch_cross_join(const CrossParams& p, hipStream_t stream) {
  const int padded = cross_padded_dim(p.dim), rows = cross_tile(padded, p.terms, p.few != 0).wq * 32;
  const dim3 grid(p.join_count, p.kv_heads);
  if (p.type == 0)
    cross_join_kernel<float><<<grid, 256, 0, stream>>>(p, padded, rows);
  else if (p.type == 1)
    cross_join_kernel<cross::bf16_t><<<grid, 256, 0, stream>>>(p, padded, rows);
  else
    cross_join_kernel<cross::half_t><<<grid, 256, 0, stream>>>(p, padded, rows);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
