// A branch's norm, its gate and residual, and the next norm with its modulation, one pass over the rows:
//   h' = post(h);  x' = c x + gate[b] h';  out = x';  normed = pre(x') (1 + scale[b]) + shift[b].
// Statistics are fp32 sums of the row's values less its first mean, whose own sum corrects that mean: a row far from
// zero keeps the precision of its differences.

#include "tsplat_common.h"
#include "tsplat_launch.h"

namespace tsplat {
namespace {

constexpr int kThreads = 256;

__device__ float block_sum(float v, float* lds) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < kThreads / 64; ++i) s += lds[i];
  return s;
}

struct Stats {
  float mean, left, inv;  // normed value = (v - mean - left) * inv
};

template <typename F>
__device__ Stats row_stats(int kind, float eps, int cols, float* lds, F value) {
  if (kind == kNormNone) return {0.0f, 0.0f, 1.0f};
  const float n = (float)cols;
  float mean = 0.0f, left = 0.0f;
  if (kind == kNormLayer) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < cols; c += kThreads) s += value(c);
    mean = block_sum(s, lds) / n;
  }
  float s = 0.0f, q = 0.0f;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float d = value(c) - mean;
    s += d;
    q = fmaf(d, d, q);
  }
  q = block_sum(q, lds) / n;
  if (kind == kNormLayer) {
    left = block_sum(s, lds) / n;
    q = fmaxf(q - left * left, 0.0f);
  }
  return {mean, left, 1.0f / sqrtf(q + eps)};
}

__device__ __forceinline__ float normed_value(const NormSpec& s, const Stats& st, float v, int c) {
  if (s.kind == kNormNone) return v;
  v = (v - st.mean - st.left) * st.inv;
  if (s.weight) v *= s.weight[c];
  if (s.bias) v += s.bias[c];
  return v;
}

// One workgroup a row of any width; the row is read again for each sum.
__global__ __launch_bounds__(kThreads) void residual_norm_row_kernel(ResidualNormParams p) {
  __shared__ float lds[kThreads / 64];
  const int64_t row = blockIdx.x, b = row / p.rows_per_batch;
  const float* x = p.x + row * p.x_stride;
  const float* h = p.h + row * p.h_stride;
  float* out = p.out + row * p.out_stride;
  float* normed = p.normed + row * p.normed_stride;
  const float* gate = p.gate ? p.gate + b * p.gate_stride : nullptr;
  const Stats post = row_stats(p.post.kind, p.post.eps, p.cols, lds, [&](int c) { return h[c]; });
  for (int c = threadIdx.x; c < p.cols; c += kThreads) {
    const float v = normed_value(p.post, post, h[c], c);
    out[c] = fmaf(p.residual_scale, x[c], gate ? gate[c] * v : v);
  }
  // (a thread reads back what it wrote itself)
  const Stats pre = row_stats(p.pre.kind, p.pre.eps, p.cols, lds, [&](int c) { return out[c]; });
  for (int c = threadIdx.x; c < p.cols; c += kThreads) {
    float v = normed_value(p.pre, pre, out[c], c);
    if (p.scale) v = fmaf(v, 1.0f + p.scale[b * p.mod_stride + c], p.shift[b * p.mod_stride + c]);
    normed[c] = v;
  }
}

}  // namespace

int launch_residual_norm(const ResidualNormParams& p, hipStream_t stream) {
  residual_norm_row_kernel<<<(unsigned)p.rows, kThreads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
