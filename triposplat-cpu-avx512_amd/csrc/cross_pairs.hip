// Cross attention of fp32 values as pairs of fp16 values, for many rows: three products of 16-bit terms where bf16 terms
// take six.
//   q' sq = qh + ql,  k sk = kh + kl,  v sv = vh + vl,  p = ph + pl
//   S = qh kh + ql kh + qh kl,  O = ph vh + pl vh + ph vl
// A pair holds its value to 2^-23 of it and to 2^-25; products of fp16 values are exact in fp32 and the dropped ones are
// below 2^-22 of the product.  sq, a power of two of the row's own, brings q's largest magnitude to [2^14, 2^15); sk and sv
// are the workgroup's and bring the largest of its first tile of states to [2^9, 2^10), so that what lies 32 times as high
// still fits and what lies 2^35 below is lost.
//
// What the pairs do not serve, and the workgroup finds while it reads the states: a magnitude of 2^15 and more of the
// scaled values (an infinity too); scores that may lose 2^-22 log2 units to the 2^-25 of k's values (|q'|_1 / sk of 8 and
// more) or of q's (D times k's largest, over sq, likewise); four neighbouring values of v, not all zero, below 2^-4, or a
// feature of v, not all zero, that stays below 2^-4 in all of the states; an infinity or NaN in q.  It then leaves its result
// to the kernel of bf16 terms, which is launched behind this one and does what is flagged, at that kernel's time.  So a value
// of v is held to 2^-23 of it or to 2^-21 of the larger of its feature's largest, over the workgroup's states, and its
// neighbours'.  (Each value by itself cannot be asked for 2^-4: one in 2000 of a normal distribution is below.)
//
// p = 2^(x - m) for a reference m that is 11 below the row's largest x, or up to 15 (few tiles rescale): below 2^15, and a
// weight 2^-36 of the largest is still held.  (The exponential's argument is rounded by 2^-21 at most there, 3e-7 of a
// weight, which its sum has as well; a factor after the exponential instead takes 16 more instructions a block.)
//
// 2 x 16384 x 2048, 16 heads of 64: 861 us (22 of them the checks by feature and key; bf16 terms 1300; the flags' launch 5),
// 0.32 PFLOP/s of the operator's operations, 0.96 of fp16 products.  A request whose first tile is masked throughout (128 states
// for heads up to 64, 32 for wider ones) has no scale from it and goes to the bf16 terms: 2150 us.  What bounds the kernel:
// products (45 % of the SIMDs' cycles) and vector instructions (52 %) that hardly overlap, as a SIMD's two waves do the same
// at the same time: waves of unlike priority, and a block's products between the exponents of the one before, did not change
// that (12 us more, and spills).
//
// Everything else as in cross_attention_kernel.h: a workgroup of eight waves of 32 rows, S^T = K Q^T, O^T = V^T P^T.

#include "cross_attention_kernel.h"

namespace tsplat {
namespace cross {

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));

constexpr float kPairSlack = 4.0f, kPairBase = 11.0f;
constexpr float kPairTop = 0x1p15f, kPairLeast = 0x1p-4f, kPairScores = 8.0f;

// Eight values as pairs.
__device__ __forceinline__ void pair8(const float (&x)[8], shortx8 (&out)[2]) {
  intx4 hi, lo;
  float minus = -1.0f;
  asm("" : "+s"(minus));  // (a product that the compiler does not turn back into two conversions and a difference)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const halfx2 h = __builtin_convertvector(floatx2{x[2 * i], x[2 * i + 1]}, halfx2);
    // (fused products take the halves where they are; exact)
    const halfx2 l = __builtin_convertvector(
        floatx2{fmaf((float)h[0], minus, x[2 * i]), fmaf((float)h[1], minus, x[2 * i + 1])}, halfx2);
    hi[i] = __builtin_bit_cast(int, h);
    lo[i] = __builtin_bit_cast(int, l);
  }
  out[0] = __builtin_bit_cast(shortx8, hi);
  out[1] = __builtin_bit_cast(shortx8, lo);
}

__device__ __forceinline__ float largest4(const float* x) {
  return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

// The exponent of the power of two that brings a magnitude to [2^top, 2^(top + 1)); 0 for zero and infinity.
__device__ __forceinline__ int exponent_to(float magnitude, int top) {
  const int e = top + 127 - (int)(__float_as_uint(magnitude) >> 23);
  return magnitude == 0.0f || !(magnitude < INFINITY) ? 0 : min(max(e, -126), 126);
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// a's and b's pairs multiplied, the small products first.
__device__ __forceinline__ floatx16 pair_products(const shortx8 (&a)[2], const shortx8 (&b)[2], floatx16 c) {
  c = multiply<half_t>(a[1], b[0], c);
  c = multiply<half_t>(a[0], b[1], c);
  return multiply<half_t>(a[0], b[0], c);
}

template <int DP, bool BIAS>
__global__ __launch_bounds__(cross_tile(DP, 3, false).wq * 64, 2) void cross_pair_kernel(CrossParams p) {
  constexpr CrossTile kTile = cross_tile(DP, 3, false);
  // (two runs of KB blocks between barriers where LDS holds them: waves that are apart multiply while others take exponents)
  constexpr int KB = kTile.kb, kRuns = DP == 64 ? 2 : 1, kWaves = kTile.wq, kThreads = kWaves * 64,
                kKeys = kRuns * KB * 32, kBlocks = DP / 32, kSlices = DP / 16;
  constexpr int kAllUnits = kKeys * DP / 8, kUnits = (kAllUnits + kThreads - 1) / kThreads;  // of 8 values
  constexpr int kRowK = DP + 8, kRowV = DP + 16;  // values from row to row
  constexpr bool kTight = DP > 96;
  constexpr int kPlaneK = kKeys * kRowK, kPlaneV = kKeys * kRowV, kBuffer = 2 * (kPlaneK + kPlaneV);
  __shared__ __attribute__((aligned(16))) short lds[2 * kBuffer];
  __shared__ __attribute__((aligned(16))) float biases[2][kKeys];
  __shared__ float largest[2][kWaves];
  __shared__ uint32_t features[DP];  // the upper bits of v's largest magnitudes
  __shared__ uint32_t k_largest;     // the bits of the scaled k's

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const Work work = work_of(p);
  const CrossItem item = p.items[work.item];
  const int kv = work.kv, D = p.dim;
  int32_t* flag = p.flags + ((int64_t)work.item * p.kv_heads + kv);

  const float* kbase = static_cast<const float*>(p.k) + (int64_t)item.key0 * p.k_token + kv * p.k_head;
  const float* vbase = static_cast<const float*>(p.v) + (int64_t)item.key0 * p.v_token + kv * p.v_head;
  const float* bias = BIAS ? p.bias + item.key0 : nullptr;
  Raw<float> kr[kUnits], vr[kUnits];
  float br[kUnits], b2 = 0.0f;
  auto load = [&](int key0) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, dim = unit % (DP / 8) * 8;
      const int64_t from = min(key0 + unit / (DP / 8), item.keys - 1);
      kr[u] = load_eight<float, true>(kbase + from * p.k_token, dim, D);
      vr[u] = load_eight<float, true>(vbase + from * p.v_token, dim, D);
      if (BIAS) br[u] = bias[from];
    }
    if (BIAS && tid < kKeys) b2 = bias[min(key0 + tid, item.keys - 1)];
  };
  // A unit's values of a tile, zeros where nothing counts.
  auto clean = [&](int u, int key0) {
    const int unit = tid + u * kThreads, dim = unit % (DP / 8) * 8;
    const bool none = key0 + unit / (DP / 8) >= item.keys || unit >= kAllUnits || (BIAS && br[u] == -INFINITY);
    kr[u] = past_end<float, true>(kr[u], dim, D, none);
    vr[u] = past_end<float, true>(vr[u], dim, D, none);
  };
  const int tiles = (item.keys + kKeys - 1) / kKeys;
  if (tiles > 0) load(0);

  // this lane's row
  const int row = wave * 32 + l32;
  const Row place = row_of(p, item, kv, row < item.rows ? row : 0);
  shortx8 q[kSlices][2];
  float from_scaled, q_sum = 0.0f;  // 1 / sq, |q'|_1: no number where q holds an infinity or NaN
  {
    Raw<float> qr[kSlices];
    const float* from = static_cast<const float*>(p.q) + place.token * p.q_token + place.head * p.q_head;
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < kSlices; ++c) {
      const int dim = 16 * c + 8 * half;
      qr[c] = past_end<float, true>(load_eight<float, true>(from, dim, D), dim, D, false);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qr[c].x[i] *= p.scale * kLog2e;
        q_sum += fabsf(qr[c].x[i]);
      }
      top = fmaxf(top, fmaxf(largest4(qr[c].x), largest4(qr[c].x + 4)));
    }
    top = fmaxf(top, other_half(top));
    q_sum += other_half(q_sum);
    const int e = exponent_to(top, 14);
    from_scaled = power(-e);
#pragma unroll
    for (int c = 0; c < kSlices; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qr[c].x[i] *= power(e);
      pair8(qr[c].x, q[c]);
    }
  }

  // the first tile's largest values, and the scales
  float k_top = 0.0f, v_top = 0.0f;
  if (tiles > 0) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      clean(u, 0);
      k_top = fmaxf(k_top, fmaxf(largest4(kr[u].x), largest4(kr[u].x + 4)));
      v_top = fmaxf(v_top, fmaxf(largest4(vr[u].x), largest4(vr[u].x + 4)));
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      k_top = fmaxf(k_top, __shfl_xor(k_top, d));
      v_top = fmaxf(v_top, __shfl_xor(v_top, d));
    }
  }
  if (lane == 0) largest[0][wave] = k_top, largest[1][wave] = v_top;
  if (tid < DP) features[tid] = 0;
  if (tid == 0) k_largest = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) k_top = fmaxf(k_top, largest[0][w]), v_top = fmaxf(v_top, largest[1][w]);
  const int ek = exponent_to(k_top, 9), ev = exponent_to(v_top, 9);
  const float k_scale = power(ek), v_scale = power(ev);
  // (never zero, which would make no number of a state past the end at -infinity; scaled scores are below 2^37, and such
  // tiny ones are zero either way)
  const float to_log2 = fmaxf(from_scaled * power(-ek), 0x1p-126f);
  bool bad = !(q_sum * power(-ek) < kPairScores);

  // Largest of the scaled k's and of v's; least: of fours of v's that are not all zero (which scaled ones may become).
  float k_most = 0.0f, v_most = 0.0f, least = INFINITY;
  // The upper 16 bits of the largest magnitudes of the eight features that this thread brings, the same in all of its units.
  static_assert(kUnits == 1 || kThreads % (DP / 8) == 0, "a thread's features");
  ushortx2 feature[4] = {};
  auto store = [&](int key0, int buf) {
    short* kp = lds + buf * kBuffer;
    short* vp = kp + 2 * kPlaneK;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, key = unit / (DP / 8), dim = unit % (DP / 8) * 8;
      if (kAllUnits % kThreads && unit >= kAllUnits) break;
      clean(u, key0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = __builtin_amdgcn_perm(__float_as_uint(vr[u].x[2 * i + 1]), __float_as_uint(vr[u].x[2 * i]),
                                                   0x07060302u) & 0x7fff7fffu;
        feature[i] = __builtin_elementwise_max(feature[i], __builtin_bit_cast(ushortx2, two));
      }
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float four = largest4(vr[u].x + i);
        v_most = fmaxf(v_most, four);
        least = fminf(least, four == 0.0f ? INFINITY : four);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) kr[u].x[i] *= k_scale, vr[u].x[i] *= v_scale;
      k_most = fmaxf(k_most, fmaxf(largest4(kr[u].x), largest4(kr[u].x + 4)));
      shortx8 kt[2], vt[2];
      pair8(kr[u].x, kt);
      pair8(vr[u].x, vt);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        *reinterpret_cast<shortx8*>(kp + t * kPlaneK + key * kRowK + dim) = kt[t];
        *reinterpret_cast<shortx8*>(vp + t * kPlaneV + key * kRowV + dim) = vt[t];
      }
    }
    if (BIAS && tid < kKeys) biases[buf][tid] = key0 + tid < item.keys ? bias_log2(b2) : -INFINITY;
  };

  floatx16 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;  // l_run: this lane's half of the row's sum
  const bool wave_live = wave * 32 < item.rows;
  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1;
    store(t * kKeys, buf);
    __syncthreads();
    if (t + 1 < tiles) load((t + 1) * kKeys);
    if (!wave_live) continue;
#pragma unroll 1
    for (int first = 0; first < kKeys; first += KB * 32) {
      if (t * kKeys + first >= item.keys) break;
      const short* kp = lds + buf * kBuffer + (first + l32) * kRowK + 8 * half;
      const short* vp = lds + buf * kBuffer + 2 * kPlaneK + (first + 4 * half + (lane & 15) / 4) * kRowV +
                        (lane >> 4 & 1) * 16 + (lane & 3) * 4;
      floatx16 s[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
        for (int c = 0; c < kSlices; ++c) {
          shortx8 kt[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            kt[i] = *reinterpret_cast<const shortx8*>(kp + i * kPlaneK + b * 32 * kRowK + 16 * c);
          s[b] = pair_products(kt, q[c], s[b]);
          in_order<kTight>();
        }
        if constexpr (BIAS) {
          const float* add = &biases[buf][first + b * 32 + 4 * half];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = fmaf(s[b][r], to_log2, add[r / 4 * 8 + r % 4]);
        } else {
          const int left = item.keys - (t * kKeys + first + b * 32) - 4 * half;  // states of this block from this lane's first
          if (left < 32) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (r / 4 * 8 + r % 4 >= left) s[b][r] = -INFINITY;
          }
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
      top = fmaxf(top, other_half(top));
      const float ref = BIAS ? top - kPairBase : fmaf(top, to_log2, -kPairBase);
      if (__any(ref > m_run + kPairSlack)) {
        const float m_new = fmaxf(m_run, ref);
        const float keep = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= keep;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[b][r] *= keep;
        m_run = m_new;
      }
      const float m = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        l_run += weights<BIAS>(s[b], to_log2, m);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = s[b][8 * c + i];
          shortx8 pt[2];
          pair8(x, pt);
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) {
            shortx8 vt[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              vt[i] = transposed(vp + i * kPlaneV + (b * 32 + 16 * c) * kRowV + 32 * d, kRowV);
            o[d] = pair_products(vt, pt, o[d]);
            in_order<kTight>();
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < 8; ++i) atomicMax(&features[tid % (DP / 8) * 8 + i], (uint32_t)feature[i / 2][i % 2]);
  atomicMax(&k_largest, __float_as_uint(k_most));
  __syncthreads();
  const float k_all = __uint_as_float(k_largest);
  bad |= !(k_all < kPairTop) || !(to_log2 * k_all * (float)D < kPairScores);
  bad |= !(v_most * v_scale < kPairTop) || least * v_scale < kPairLeast;
  if (tid < DP && features[tid] != 0) bad |= __uint_as_float(features[tid] << 16) * v_scale < kPairLeast;
  bad = __syncthreads_or(bad);
  if (tid == 0) *flag = bad;
  const int again = thread_again(), out_row = (again >> 6) * 32 + (again & 31);
  if (bad || out_row >= item.rows) return;
  // Weights of 1 at most before v's scale is undone: sums that fp32 holds stay within it.
  constexpr float kMost = kPairBase + kPairSlack, kDown = 1.0f / (1 << (int)kMost);
  const float l = (l_run + other_half(l_run)) * kDown, down = power(-ev);
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = o[b][r] * kDown * down;
  finish<float, DP, true>(p, item, kv, out_row, kWaves * 32, row_of(p, item, kv, out_row), again >> 5 & 1, o,
                          m_run + kMost, l);
}

template <int DP>
int launch_pairs(const CrossParams& p, hipStream_t stream) {
  const int grid = p.item_count * p.kv_heads, threads = cross_tile(DP, 3, false).wq * 64;
  if (p.bias)
    cross_pair_kernel<DP, true><<<grid, threads, 0, stream>>>(p);
  else
    cross_pair_kernel<DP, false><<<grid, threads, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace cross

int launch_cross_pairs(const CrossParams& p, hipStream_t stream) {
  switch (cross_padded_dim(p.dim)) {
    case 64: return cross::launch_pairs<64>(p, stream);
    case 96: return cross::launch_pairs<96>(p, stream);
    default: return cross::launch_pairs<128>(p, stream);
  }
}

}  // namespace tsplat
