// Rotary positions of several axes, the per-head RMS norm and the attention's layout in one pass:
//   (a, b) of pair p -> (a cos t - b sin t, a sin t + b cos t),  t = 2 pi positions[axis[p]] turns[p],
//   z = y sqrt(D) / max(||y||, eps) gamma[h]     (||y|| = ||x||: a rotation keeps it).
// The angle is taken in revolutions and in 64 bits, where only its fraction counts: a far position keeps the
// precision that its fp32 product with a frequency would lose.  8 bytes a value from and to HBM, which bounds it.

#include <algorithm>
#include <type_traits>

#include "tsplat_common.h"
#include "tsplat_launch.h"
#include "wave_sum.h"

namespace tsplat {
namespace {

typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));  // vectors start at any float

// A workgroup: kTokenWaves waves along the tokens, each with kVectorWaves shares of their parts' heads.  16384 tokens x
// 16 x 64, q, k and v: 87 us, 4.6 TB/s (a copy of as much: 73-79); one token wave with 4 shares 94-110 (writes of 2 KiB
// a head instead of 8).
constexpr int kTokenWaves = 4, kVectorWaves = 4, kThreads = kTokenWaves * kVectorWaves * 64;
constexpr int kAhead = 2;  // vectors that a lane asks for at once (with one token wave 4: 107 us, 2: 112, 1: 94)

// G lanes a vector, lane i of them its pairs 4 i .. 4 i + 3; the last one with any takes the vector's last four, some of
// which its neighbour has too and writes alike (28899 x 3 x 182: 38 us, 63 with single values there, which all lanes
// wait for).  A wave turns 64 / G tokens.  The workgroup computes its tokens' sines and cosines once, into LDS, and a
// lane keeps its own while it goes through its share of the vectors.  64 registers let two workgroups share a compute
// unit (without that bound neighbours take 84: 1640 x 17 x 150, q, k and v, 35 us, so 26).
template <int G, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads, 8) void rope_axes_kernel(RopeAxesParams p) {
  constexpr int kTokens = 64 / G, kAllTokens = kTokens * kTokenWaves;
  __shared__ float2 circle[kAllTokens * G * 4];
  // (the wave's number as a scalar, so that what follows from it is one too)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tokens = (int64_t)p.B * p.L;
  const int64_t token0 = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * kAllTokens;
  const int64_t token = token0 + wave / kVectorWaves * kTokens + lane / G;
  const int share = blockIdx.x * kVectorWaves + wave % kVectorWaves, shares = gridDim.x * kVectorWaves;
  const int pairs = p.D / 2, vectors = p.parts * p.H;
  for (uint32_t i = threadIdx.x; i < (uint32_t)(kAllTokens * pairs); i += kThreads) {
    const uint32_t t = i / (uint32_t)pairs, pair = i - t * (uint32_t)pairs;
    if (token0 + t >= tokens) break;
    const uint32_t b = (uint32_t)(token0 + t) / (uint32_t)p.L, l = (uint32_t)(token0 + t) - b * (uint32_t)p.L;
    int axis = p.axis[pair];
    if (axis < 0 || axis >= p.axes) axis = 0;
    const int64_t at = ((int64_t)(p.position_batches > 1 ? b : 0) * p.L + l) * p.axes + axis;
    const double pos = p.position_type ? (double)static_cast<const float*>(p.positions)[at]
                                       : (double)static_cast<const int32_t*>(p.positions)[at];
    const double turn = pos * p.turns[pair];
    float2 v;
    sincospif(2.0f * (float)(turn - rint(turn)), &v.y, &v.x);
    circle[t * G * 4 + pair] = v;
  }
  __syncthreads();
  const int own = lane % G * 4, i0 = max(0, min(own, pairs - 4));
  const int n = token < tokens && own < pairs ? min(4, pairs) : 0;  // pairs of this lane
  const int twice = own - i0;                                       // the first ones of them, which a neighbour has too
  // (tokens are fewer than 2^31: a division of 32 bits takes a fifth of one of 64)
  const uint32_t live = token < tokens ? (uint32_t)token : 0;
  const uint32_t b = live / (uint32_t)p.L, l = live - b * (uint32_t)p.L;
  float cs[4], sn[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = e < n ? circle[(int)(token - token0) * G * 4 + i0 + e] : make_float2(1.0f, 0.0f);
    cs[e] = v.x;
    sn[e] = v.y;
  }
  const float root = sqrtf((float)p.D);
  // element offsets of the pairs' first and second values: 8 neighbours, or 4 of each half
  const int j0 = INTERLEAVED ? 2 * i0 : i0, j1 = INTERLEAVED ? 2 * i0 + 4 : i0 + pairs;
  const float* src = p.x + b * p.batch_stride + l * p.token_stride;
  const int64_t dst = (p.out_bhld ? (int64_t)b * p.H * p.L + l : (int64_t)live * p.H) * p.D;
  const int64_t dst_head = (p.out_bhld ? (int64_t)p.L : 1) * p.D;
  const bool few = G == 1 && pairs < 4;
  // (lanes without a token or pairs load others')
  auto load = [&](const float* v, floatx4& lo, floatx4& hi) {
    if (!few) {
      lo = *reinterpret_cast<const floatx4u*>(v + j0);
      hi = *reinterpret_cast<const floatx4u*>(v + j1);
    } else {
      lo = hi = floatx4{};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (INTERLEAVED) {
          if (e < 2 * n) lo[e] = v[j0 + e];
          if (e + 4 < 2 * n) hi[e] = v[j1 + e];
        } else if (e < n) {
          lo[e] = v[j0 + e];
          hi[e] = v[j1 + e];
        }
      }
    }
  };
  auto store = [&](float* v, const floatx4& lo, const floatx4& hi) {
    if (!few) {
      *reinterpret_cast<floatx4u*>(v + j0) = lo;
      *reinterpret_cast<floatx4u*>(v + j1) = hi;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (INTERLEAVED) {
          if (e < 2 * n) v[j0 + e] = lo[e];
          if (e + 4 < 2 * n) v[j1 + e] = hi[e];
        } else if (e < n) {
          v[j0 + e] = lo[e];
          v[j1 + e] = hi[e];
        }
      }
    }
  };
  for (int first = share; first < vectors; first += shares * kAhead) {
    floatx4 lo[kAhead], hi[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = first + u * shares;
      if (v < vectors) load(src + (v / p.H) * p.part_stride + (v % p.H) * p.head_stride, lo[u], hi[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = first + u * shares;
      if (v >= vectors) break;  // the same for the whole wave
      const int part = v / p.H, h = v % p.H;
      floatx4 a = lo[u], c = hi[u];
      if (part < 2) {
        const float* gamma = p.gamma[part];
        float scale = 1.0f;
        floatx4 g0, g1;
        if (gamma) {
          load(gamma + (int64_t)h * p.D, g0, g1);
          float q = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float re = INTERLEAVED ? (e < 2 ? a[2 * e] : c[2 * e - 4]) : a[e];
            const float im = INTERLEAVED ? (e < 2 ? a[2 * e + 1] : c[2 * e - 3]) : c[e];
            q += e < twice ? 0.0f : fmaf(re, re, im * im);
          }
          const float norm = sqrtf(group_sum<G>(q));
          scale = root / (norm < p.eps ? p.eps : norm);  // (a NaN stays one, which fmaxf would hide from its neighbours)
        }
        floatx4 y0, y1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (INTERLEAVED) {
            const float re = e < 2 ? a[2 * e] : c[2 * e - 4], im = e < 2 ? a[2 * e + 1] : c[2 * e - 3];
            const float t0 = re * cs[e] - im * sn[e], t1 = re * sn[e] + im * cs[e];
            if (e < 2)
              y0[2 * e] = t0, y0[2 * e + 1] = t1;
            else
              y1[2 * e - 4] = t0, y1[2 * e - 3] = t1;
          } else {
            y0[e] = a[e] * cs[e] - c[e] * sn[e];
            y1[e] = a[e] * sn[e] + c[e] * cs[e];
          }
        }
        if (gamma) {
          y0 = y0 * scale * g0;
          y1 = y1 * scale * g1;
        }
        a = y0;
        c = y1;
      }
      if (n > 0) store(p.out[part] + h * dst_head + dst, a, c);
    }
  }
}

}  // namespace

int launch_rope_axes(const RopeAxesParams& p, hipStream_t stream) {
  const int lanes = (p.D / 2 + 3) / 4;
  auto run = [&](auto g) {
    constexpr int G = decltype(g)::value;
    const int64_t tokens = (int64_t)p.B * p.L, groups = (tokens + 64 / G * kTokenWaves - 1) / (64 / G * kTokenWaves);
    // four vectors a wave; fewer where few tokens leave the chip idle
    const int vectors = p.parts * p.H;
    const int64_t blocks = std::min<int64_t>((vectors + kVectorWaves - 1) / kVectorWaves,
                                             std::max<int64_t>((vectors + 4 * kVectorWaves - 1) / (4 * kVectorWaves),
                                                               512 / groups));
    const int64_t row = std::min<int64_t>(groups, 65535);
    const dim3 grid((unsigned)blocks, (unsigned)row, (unsigned)((groups + row - 1) / row));
    if (p.interleaved)
      rope_axes_kernel<G, true><<<grid, kThreads, 0, stream>>>(p);
    else
      rope_axes_kernel<G, false><<<grid, kThreads, 0, stream>>>(p);
  };
  if (lanes <= 1)
    run(std::integral_constant<int, 1>{});
  else if (lanes <= 2)
    run(std::integral_constant<int, 2>{});
  else if (lanes <= 4)
    run(std::integral_constant<int, 4>{});
  else if (lanes <= 8)
    run(std::integral_constant<int, 8>{});
  else if (lanes <= 16)
    run(std::integral_constant<int, 16>{});
  else if (lanes <= 32)
    run(std::integral_constant<int, 32>{});
  else
    run(std::integral_constant<int, 64>{});
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
