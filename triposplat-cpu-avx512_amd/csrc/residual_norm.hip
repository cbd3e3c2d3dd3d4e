// A branch's norm, its gate and residual, and the next norm with its modulation, one pass over the rows:
//   h' = post(h);  x' = c x + gate[b] h';  out = x';  normed = pre(x') (1 + scale[b]) + shift[b].
// 16 bytes a value from and to HBM, which bounds it: 12294 x 1024 38 us (5.3 TB/s), 8202 x 4096 with both norms 94 us
// (5.7).  A row stays in registers from the first load to the last store: in those of 8, 16 or 32 lanes up to 32, 64 or
// 128 columns (a wave a row there: 339832 x 39 106 us, so 34; 37899 x 77 25, so 16), of one wave up to 2048, of four up
// to 8192 (at 2048 columns the two are alike, 50 us for 7812 rows).
// Statistics are fp32 sums of the row's values less its first mean, whose own sum corrects that mean: a row far from
// zero keeps the precision of its differences.

#include <algorithm>
#include <type_traits>

#include "tsplat_common.h"
#include "tsplat_launch.h"
#include "wave_sum.h"

namespace tsplat {
namespace {

typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any float

__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// The sum over the R lanes of a row, in each of them.  lds: a float a wave for each call that may be in flight.
template <int R>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  v = group_sum<std::min(R, 64)>(v);
  if constexpr (R > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < R / 64; ++i) v += lds[i];
  }
  return v;
}

struct Stats {
  float mean, left, inv;  // normed value = (v - mean - left) * inv
};

// A row in registers: R lanes, lane l of them holding columns 4 (R i + l) .. + 3 for i < V.  All but the last i
// are whole; `last` is how many of that one's four columns exist.
template <int R, int V>
struct Row {
  floatx4 v[V];
};

template <int R, int V>
__device__ __forceinline__ void load_row(Row<R, V>& r, const float* src, int c0, int last) {
#pragma unroll
  for (int i = 0; i < V - 1; ++i) r.v[i] = *reinterpret_cast<const floatx4u*>(src + c0 + i * 4 * R);
  const float* tail = src + c0 + (V - 1) * 4 * R;
  if (last >= 4) {
    r.v[V - 1] = *reinterpret_cast<const floatx4u*>(tail);
  } else {
    r.v[V - 1] = floatx4{};
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < last) r.v[V - 1][e] = tail[e];
  }
}

template <int R, int V>
__device__ __forceinline__ void store_row(const Row<R, V>& r, float* dst, int c0, int last) {
#pragma unroll
  for (int i = 0; i < V - 1; ++i) *reinterpret_cast<floatx4u*>(dst + c0 + i * 4 * R) = r.v[i];
  float* tail = dst + c0 + (V - 1) * 4 * R;
  if (last >= 4) {
    *reinterpret_cast<floatx4u*>(tail) = r.v[V - 1];
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < last) tail[e] = r.v[V - 1][e];
  }
}

// lds: 3 floats a wave.
template <int R, int V>
__device__ __forceinline__ Stats row_stats(const Row<R, V>& r, int kind, float eps, float n, int last, float* lds) {
  if (kind == kNormNone) return {0.0f, 0.0f, 1.0f};
  float mean = 0.0f, left = 0.0f;
  if (kind == kNormLayer) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += (r.v[i][0] + r.v[i][1]) + (r.v[i][2] + r.v[i][3]);  // (zeros past the end)
    mean = row_sum<R>(s, lds) / n;
  }
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = i == V - 1 && e >= last ? 0.0f : r.v[i][e] - mean;
      s += d;
      q = fmaf(d, d, q);
    }
  q = row_sum<R>(q, lds + R / 64) / n;
  if (kind == kNormLayer) {
    left = row_sum<R>(s, lds + R / 64 * 2) / n;
    q = fmaxf(q - left * left, 0.0f);
  }
  return {mean, left, 1.0f / sqrtf(q + eps)};
}

// R lanes a row, 256 / R rows a workgroup; a row's x, h, gate and modulation are all asked for at once.
template <int R, int V>
__global__ __launch_bounds__(256) void residual_norm_kernel(ResidualNormParams p) {
  __shared__ float lds[R <= 64 ? 1 : 6 * R / 64];
  int within = threadIdx.x / R;
  if (R == 64) within = __builtin_amdgcn_readfirstlane(within);  // (a scalar, so that what follows from the row is one too)
  const int64_t row = block_index() * (256 / R) + within;
  if (row >= p.rows) return;  // all lanes of a row; where they meet at barriers the whole workgroup
  const int c0 = threadIdx.x % R * 4, last = p.cols - c0 - (V - 1) * 4 * R;
  const int64_t b = p.gate || p.scale ? (uint32_t)row / (uint32_t)p.rows_per_batch : 0;
  const float n = (float)p.cols;
  Row<R, V> x, h, gate;
  load_row(h, p.h + row * p.h_stride, c0, last);
  load_row(x, p.x + row * p.x_stride, c0, last);
  if (p.gate) load_row(gate, p.gate + b * p.gate_stride, c0, last);
  // a norm's vectors are asked for before its sums, which take their time
  auto norm = [&](Row<R, V>& r, const NormSpec& s, float* sums) {
    if (s.kind == kNormNone) return;
    Row<R, V> w, bias;
    if (s.weight) load_row(w, s.weight, c0, last);
    if (s.bias) load_row(bias, s.bias, c0, last);
    const Stats st = row_stats(r, s.kind, s.eps, n, last, sums);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) r.v[i][e] = (r.v[i][e] - st.mean - st.left) * st.inv;
    if (s.weight) {
#pragma unroll
      for (int i = 0; i < V; ++i) r.v[i] *= w.v[i];
    }
    if (s.bias) {
#pragma unroll
      for (int i = 0; i < V; ++i) r.v[i] += bias.v[i];
    }
  };
  norm(h, p.post, lds);
  if (p.gate) {
#pragma unroll
    for (int i = 0; i < V; ++i) h.v[i] *= gate.v[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)  // (past the end the statistics want zeros)
      x.v[i][e] = i == V - 1 && e >= last ? 0.0f : fmaf(p.residual_scale, x.v[i][e], h.v[i][e]);
  store_row(x, p.out + row * p.out_stride, c0, last);
  Row<R, V> scale, shift;
  if (p.scale) {
    load_row(scale, p.scale + b * p.mod_stride, c0, last);
    load_row(shift, p.shift + b * p.mod_stride, c0, last);
  }
  norm(x, p.pre, lds + R / 64 * (R > 64 ? 3 : 0));
  if (p.scale) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v[i][e] = fmaf(x.v[i][e], 1.0f + scale.v[i][e], shift.v[i][e]);
  }
  store_row(x, p.normed + row * p.normed_stride, c0, last);
}

// Rows too wide for registers: one workgroup a row, which is read again for each sum (1302 x 12288: 93 us, 2.8 TB/s at
// one pass' bytes; 174 with both norms).
constexpr int kWideThreads = 1024;

__device__ float block_sum(float v, float* lds) {
  __syncthreads();  // (the sums before have been read)
  return row_sum<kWideThreads>(v, lds);
}

template <typename F>
__device__ Stats wide_stats(int kind, float eps, uint32_t cols, float* lds, F value) {
  if (kind == kNormNone) return {0.0f, 0.0f, 1.0f};
  const float n = (float)cols;
  float mean = 0.0f, left = 0.0f;
  if (kind == kNormLayer) {
    float s = 0.0f;
    for (uint32_t c = threadIdx.x; c < cols; c += kWideThreads) s += value(c);
    mean = block_sum(s, lds) / n;
  }
  float s = 0.0f, q = 0.0f;
  for (uint32_t c = threadIdx.x; c < cols; c += kWideThreads) {
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

__device__ __forceinline__ float wide_value(const NormSpec& s, const Stats& st, float v, uint32_t c) {
  if (s.kind == kNormNone) return v;
  v = (v - st.mean - st.left) * st.inv;
  if (s.weight) v *= s.weight[c];
  if (s.bias) v += s.bias[c];
  return v;
}

__global__ __launch_bounds__(kWideThreads) void residual_norm_wide_kernel(ResidualNormParams p) {
  __shared__ float lds[kWideThreads / 64];
  const int64_t row = block_index();
  if (row >= p.rows) return;
  const uint32_t cols = (uint32_t)p.cols;  // (a column past the last one may pass 2^31)
  const int64_t b = p.gate || p.scale ? (uint32_t)row / (uint32_t)p.rows_per_batch : 0;
  const float* x = p.x + row * p.x_stride;
  const float* h = p.h + row * p.h_stride;
  float* out = p.out + row * p.out_stride;
  float* normed = p.normed + row * p.normed_stride;
  const float* gate = p.gate ? p.gate + b * p.gate_stride : nullptr;
  const Stats post = wide_stats(p.post.kind, p.post.eps, cols, lds, [&](uint32_t c) { return h[c]; });
  for (uint32_t c = threadIdx.x; c < cols; c += kWideThreads) {
    const float v = wide_value(p.post, post, h[c], c);
    out[c] = fmaf(p.residual_scale, x[c], gate ? gate[c] * v : v);
  }
  // (a thread reads back what it wrote itself)
  const Stats pre = wide_stats(p.pre.kind, p.pre.eps, cols, lds, [&](uint32_t c) { return out[c]; });
  for (uint32_t c = threadIdx.x; c < cols; c += kWideThreads) {
    float v = wide_value(p.pre, pre, out[c], c);
    if (p.scale) v = fmaf(v, 1.0f + p.scale[b * p.mod_stride + c], p.shift[b * p.mod_stride + c]);
    normed[c] = v;
  }
}

dim3 grid_of(int64_t blocks) {
  const int64_t x = std::min<int64_t>(blocks, 1 << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

template <int R, int V>
void launch_row(const ResidualNormParams& p, hipStream_t stream) {
  residual_norm_kernel<R, V><<<grid_of((p.rows + 256 / R - 1) / (256 / R)), 256, 0, stream>>>(p);
}

template <int R>
void launch_rows(const ResidualNormParams& p, hipStream_t stream) {
  const int chunks = (p.cols + 4 * R - 1) / (4 * R);
  if constexpr (R == 64) {  // (wider rows have three chunks at least)
    if (chunks == 1) return launch_row<R, 1>(p, stream);
    if (chunks == 2) return launch_row<R, 2>(p, stream);
  }
  switch (chunks) {
    case 3: launch_row<R, 3>(p, stream); break;
    case 4: launch_row<R, 4>(p, stream); break;
    case 5: launch_row<R, 5>(p, stream); break;
    case 6: launch_row<R, 6>(p, stream); break;
    case 7: launch_row<R, 7>(p, stream); break;
    default: launch_row<R, 8>(p, stream); break;
  }
}

}  // namespace

int launch_residual_norm(const ResidualNormParams& p, hipStream_t stream) {
  if (p.cols <= 32)
    launch_row<8, 1>(p, stream);
  else if (p.cols <= 64)
    launch_row<16, 1>(p, stream);
  else if (p.cols <= 128)
    launch_row<32, 1>(p, stream);
  else if (p.cols <= 2048)
    launch_rows<64>(p, stream);
  else if (p.cols <= 8192)
    launch_rows<256>(p, stream);
  else
    residual_norm_wide_kernel<<<grid_of(p.rows), kWideThreads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
