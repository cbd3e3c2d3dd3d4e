// Rotary positions of several axes, the per-head RMS norm and the attention's layout in one pass:
//   (a, b) of pair p -> (a cos t - b sin t, a sin t + b cos t),  t = 2 pi positions[axis[p]] turns[p],
//   z = y sqrt(D) / max(||y||, eps) gamma[h].
// The angle is taken in revolutions and in 64 bits, where only its fraction counts: a far position keeps the
// precision that its fp32 product with a frequency would lose.

#include "tsplat_common.h"
#include "tsplat_launch.h"

namespace tsplat {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;

// One workgroup a token, one wave a head's vector.
__global__ __launch_bounds__(kThreads) void rope_axes_token_kernel(RopeAxesParams p) {
  __shared__ float cos_lds[kMaxPairs], sin_lds[kMaxPairs];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t token = blockIdx.x;
  const int64_t b = token / p.L, l = token % p.L;
  const int pairs = p.D / 2;
  for (int i = tid; i < pairs; i += kThreads) {
    int axis = p.axis[i];
    if (axis < 0 || axis >= p.axes) axis = 0;
    const int64_t at = ((p.position_batches > 1 ? b : 0) * p.L + l) * p.axes + axis;
    const double pos = p.position_type ? (double)static_cast<const float*>(p.positions)[at]
                                       : (double)static_cast<const int32_t*>(p.positions)[at];
    const double t = pos * p.turns[i];
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    cos_lds[i] = c;
    sin_lds[i] = s;
  }
  __syncthreads();
  for (int v = wave; v < p.parts * p.H; v += kThreads / 64) {
    const int part = v / p.H, h = v % p.H;
    const float* src = p.x + part * p.part_stride + b * p.batch_stride + l * p.token_stride + h * p.head_stride;
    float* dst = p.out[part] + (p.out_bhld ? (b * p.H + h) * p.L + l : (b * p.L + l) * p.H + h) * p.D;
    if (part == 2) {
      for (int d = lane; d < p.D; d += 64) dst[d] = src[d];
      continue;
    }
    const float* gamma = p.gamma[part] ? p.gamma[part] + h * p.D : nullptr;
    float scale = 1.0f;
    if (gamma) {
      float q = 0.0f;
      for (int d = lane; d < p.D; d += 64) q = fmaf(src[d], src[d], q);
      for (int d = 32; d; d >>= 1) q += __shfl_xor(q, d);
      scale = sqrtf((float)p.D) / fmaxf(sqrtf(q), p.eps);
    }
    for (int i = lane; i < pairs; i += 64) {
      const int j0 = p.interleaved ? 2 * i : i, j1 = p.interleaved ? 2 * i + 1 : i + pairs;
      const float a0 = src[j0], a1 = src[j1], c = cos_lds[i], s = sin_lds[i];
      const float y0 = a0 * c - a1 * s, y1 = a0 * s + a1 * c;
      dst[j0] = gamma ? y0 * scale * gamma[j0] : y0;
      dst[j1] = gamma ? y1 * scale * gamma[j1] : y1;
    }
  }
}

}  // namespace

int launch_rope_axes(const RopeAxesParams& p, hipStream_t stream) {
  rope_axes_token_kernel<<<p.B * p.L, kThreads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
