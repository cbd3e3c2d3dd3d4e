// Low-rank adapters of many requests beside a shared Linear:
//   out[m] = y[m] + scale[a] (x[m] down[a]^T) up[a]^T,  a = rows[m].
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "tsplat_common.h"
#include "tsplat_launch.h"

namespace tsplat {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRank = 512;

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float value_of(__half v) { return __half2float(v); }

// One workgroup a row: its inner values in LDS, then its outputs.
template <typename T>
__global__ __launch_bounds__(kThreads) void low_rank_row_kernel(LowRankParams p) {
  __shared__ float inner[kMaxRank];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.x;
  const float* y = p.y + m * p.y_stride;
  float* out = p.out + m * p.out_stride;
  const int a = p.rows[m];
  const int rank = a >= 0 && a < p.slots ? min(p.rank[a], p.R) : 0;
  if (rank <= 0) {
    if (p.out != p.y)
      for (int n = tid; n < p.N; n += kThreads) out[n] = y[n];
    return;
  }
  const float* x = p.x + m * p.x_stride;
  const int k_tiles = (p.K + 31) / 32, r_tiles = (p.R + 15) / 16, n_tiles = (p.N + 15) / 16, r_steps = (p.R + 31) / 32;
  const T* down = static_cast<const T*>(p.down) + (int64_t)a * r_tiles * k_tiles * 512;
  const T* up = static_cast<const T*>(p.up) + (int64_t)a * n_tiles * r_steps * 512;
  for (int r = wave; r < rank; r += kThreads / 64) {
    float sum = 0.0f;
    for (int k = lane; k < p.K; k += 64)
      sum = fmaf(x[k], value_of(down[((int64_t)(r >> 4) * k_tiles + (k >> 5)) * 512 + ((k >> 3) & 3) * 128 +
                                     (r & 15) * 8 + (k & 7)]),
                 sum);
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) inner[r] = sum * p.scale[a];
  }
  __syncthreads();
  for (int n = tid; n < p.N; n += kThreads) {
    float sum = 0.0f;
    for (int r = 0; r < rank; ++r)
      sum = fmaf(inner[r], value_of(up[((int64_t)(n >> 4) * r_steps + (r >> 5)) * 512 + ((r >> 3) & 3) * 128 +
                                       (n & 15) * 8 + (r & 7)]),
                 sum);
    out[n] = y[n] + sum;
  }
}

}  // namespace

int64_t low_rank_scratch_bytes(int, int, int, int, int, int) { return 0; }

int launch_low_rank_add(const LowRankParams& p, hipStream_t stream) {
  switch (p.dtype) {
    case kAdapterF32: low_rank_row_kernel<float><<<p.M, kThreads, 0, stream>>>(p); break;
    case kAdapterBf16: low_rank_row_kernel<__hip_bfloat16><<<p.M, kThreads, 0, stream>>>(p); break;
    default: low_rank_row_kernel<__half><<<p.M, kThreads, 0, stream>>>(p); break;
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
