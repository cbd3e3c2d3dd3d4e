// Cross attention of a batch of requests, each query row over its own request's states:
//   out = sum_j softmax_j(scale q . k_j + bias_j) v_j,
// one pass over the states with the running maximum and sum of the softmax.
//
// A wave owns 32 rows (query token x head of the key head's group) and computes S^T = K Q^T, 32 states at a time: a lane
// then holds 16 states of one row, so a row's maximum and sum are in-lane steps and one swap of half waves, and P^T is the
// second product's operand as it stands.  O^T = V^T P^T: V^T comes out of LDS by the transposing reads, four states of 16
// columns each, in the order that the first product's accumulators hold them (state 8 (r / 4) + 4 (lane / 32) + r % 4 in
// register r).
// 16-bit values are multiplied as they are, the probabilities rounded to the values' type (each by half a step, below
// the rounding of the result).  fp32 values are split into TERMS bf16 terms: 3 keep all 24 bits (the six products above
// 2^-24 of the largest are added, smallest first), 2 keep 16 bits (three products), 1 rounds to bf16; scale and log2 e
// are multiplied into q before.  Sums, maxima and exponents are fp32.
//
// States go from memory through registers to LDS, a tile ahead of the products; states that the bias masks, or past the
// request's last, are put there as zeros, so what memory holds in their place does not matter.  Rows of LDS are padded so
// that eight rows (K, 16 bytes of each) and four rows (V, 32 bytes of each) fall into different banks.
#pragma once

#include <type_traits>

#include "cross_attention.h"
#include "tsplat_common.h"

namespace tsplat {
namespace cross {

typedef __bf16 bf16_t;
typedef _Float16 half_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
// Weights are 2^(x - m) for a reference m that follows a row's largest x (log2 units) only when that has passed it by more
// than kSlack: most tiles rescale nothing.  fp16 weights lie 2^7 higher, below 2^15 at most, so that a weight 2^-31 of the
// largest is still held (many small ones add up); bf16 has fp32's range.
constexpr float kSlack = 8.0f;
template <class E>
constexpr float kLift = std::is_same_v<E, half_t> ? 7.0f : 0.0f;

template <class T>
struct Element {
  typedef bf16_t type;
};
template <>
struct Element<half_t> {
  typedef half_t type;
};

template <class E>
__device__ __forceinline__ floatx16 multiply(const shortx8& a, const shortx8& b, const floatx16& c) {
  if constexpr (std::is_same_v<E, half_t>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Pairs of values to 16 bits, nearest even; `left` what is left of them (exact).
__device__ __forceinline__ int bf16_pair(float a, float b, float& left_a, float& left_b) {
  const int w = __builtin_bit_cast(int, bf16x2{(bf16_t)a, (bf16_t)b});
  left_a = a - __int_as_float(w << 16);
  left_b = b - __int_as_float(w & 0xffff0000);
  return w;
}

// Eight values as TERMS vectors of 16-bit terms.
template <class E, int TERMS>
__device__ __forceinline__ void split8(const float (&x)[8], shortx8 (&out)[TERMS]) {
  if constexpr (std::is_same_v<E, half_t>) {
    halfx8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (half_t)x[i];
    out[0] = __builtin_bit_cast(shortx8, h);
  } else {
    float left[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] = x[i];
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      intx4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        w[i] = bf16_pair(left[2 * i], left[2 * i + 1], a, b);
        left[2 * i] = a, left[2 * i + 1] = b;
      }
      out[t] = __builtin_bit_cast(shortx8, w);
    }
  }
}

// Eight values of a row from dim on, as they are in memory; zero past the vector's end.
template <class T>
struct Raw {
  T x[8];
};
template <class T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int dim, int D, bool vec) {
  Raw<T> r;
  if (vec) {
    if (dim < D)
      __builtin_memcpy(&r, __builtin_assume_aligned(row + dim, 16), sizeof(r));
    else
      __builtin_memset(&r, 0, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = dim + i < D ? row[dim + i] : (T)0.0f;
  }
  return r;
}

// The terms of eight values; of T's own 16 bits as they are.
template <class T, class E, int TERMS>
__device__ __forceinline__ void terms_of(const Raw<T>& r, shortx8 (&out)[TERMS]) {
  if constexpr (sizeof(T) == 2) {
    out[0] = __builtin_bit_cast(shortx8, r);
  } else {
    split8<E, TERMS>(r.x, out);
  }
}

__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return (threadIdx.x & 32) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}

// a's and b's terms multiplied, the small products first.
template <class E, int TERMS>
__device__ __forceinline__ floatx16 products(const shortx8 (&a)[TERMS], const shortx8 (&b)[TERMS], floatx16 c) {
#pragma unroll
  for (int sum = TERMS - 1; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i) c = multiply<E>(a[sum - i], b[i], c);
  return c;
}

template <class T, int TERMS, int DP, bool FEW, bool BIAS>
__global__ __launch_bounds__(cross_tile(DP, TERMS, FEW).wq* cross_tile(DP, TERMS, FEW).wk * 64) void cross_kernel(
    CrossParams p) {
  typedef typename Element<T>::type E;
  constexpr CrossTile kTile = cross_tile(DP, TERMS, FEW);
  constexpr int WQ = kTile.wq, WK = kTile.wk, KB = kTile.kb, BUFS = kTile.bufs;
  constexpr int kThreads = WQ * WK * 64, kKeys = WK * KB * 32, kBlocks = DP / 32, kSlices = DP / 16;
  constexpr int kAllUnits = kKeys * DP / 8, kUnits = (kAllUnits + kThreads - 1) / kThreads;  // of 8 values
  constexpr int kRowK = DP + 8, kRowV = DP + 16;  // values from row to row
  constexpr int kPlaneK = kKeys * kRowK, kPlaneV = kKeys * kRowV;
  constexpr int kBuffer = TERMS * (kPlaneK + kPlaneV);
  constexpr int kMerge = (WK - 1) * WQ * (DP / 2 + 2) * 64 * 2;  // shorts of the waves' sums that meet at the end
  constexpr int kLds = BUFS * kBuffer > kMerge ? BUFS * kBuffer : kMerge;
  __shared__ __attribute__((aligned(16))) short lds[kLds];
  __shared__ float biases[BUFS][kKeys];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave / WK, wk = wave % WK;
  const int l32 = lane & 31, half = lane >> 5;
  // neighbours on an XCD share a key head
  const int count = gridDim.x, per = count / 8, more = count % 8, xcd = blockIdx.x % 8;
  const int id = xcd * per + min(xcd, more) + blockIdx.x / 8;
  const CrossItem item = p.items[id % p.item_count];
  const int kv = id / p.item_count;
  const bool vec = p.vec;
  const int D = p.dim;

  // this lane's row
  const int row = wq * 32 + l32;
  const bool live = row < item.rows;
  const int at = item.row0 + (live ? row : 0);
  const int64_t token = item.token0 + at / p.group;
  const int head = kv * p.group + at % p.group;

  // Q: columns 16 c + 8 half + i of the row in slice c
  shortx8 q[kSlices][TERMS];
  const T* qrow = static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head;
#pragma unroll
  for (int c = 0; c < kSlices; ++c) {
    Raw<T> r = load_raw<T>(qrow, 16 * c + 8 * half, D, vec);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.x[i] *= p.scale * kLog2e;
    }
    terms_of<T, E, TERMS>(r, q[c]);
  }
  const float to_log2 = sizeof(T) == 4 ? 1.0f : p.scale * kLog2e;

  const T* kbase = static_cast<const T*>(p.k) + (int64_t)item.key0 * p.k_token + kv * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + (int64_t)item.key0 * p.v_token + kv * p.v_head;
  const float* bias = p.bias + (BIAS ? item.key0 : 0);

  Raw<T> kr[kUnits], vr[kUnits];
  uint32_t masked = 0;  // a bit for each unit
  float b2 = 0.0f;
  auto load = [&](int key0) {
    masked = 0;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, key = key0 + unit / (DP / 8), dim = unit % (DP / 8) * 8;
      const bool real = key < item.keys && unit < kAllUnits;
      const int64_t from = real ? key : 0;
      kr[u] = load_raw<T>(kbase + from * p.k_token, dim, D, vec);
      vr[u] = load_raw<T>(vbase + from * p.v_token, dim, D, vec);
      if (!real || (BIAS && bias[from] == -INFINITY)) masked |= 1u << u;
    }
    if (BIAS && tid < kKeys) {
      // log2 units; a finite bias stays finite (the type's lowest masks against others, not by itself)
      const float b = key0 + tid < item.keys ? bias[key0 + tid] : -INFINITY;
      b2 = b == -INFINITY ? b : fmaxf(b * kLog2e, -3.4028234663852886e38f);
      if (b != b) b2 = b;
    }
  };
  auto store = [&](int buf) {
    short* kp = lds + buf * kBuffer;
    short* vp = kp + TERMS * kPlaneK;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, key = unit / (DP / 8), dim = unit % (DP / 8) * 8;
      if (kAllUnits % kThreads && unit >= kAllUnits) break;
      shortx8 kt[TERMS], vt[TERMS];
      terms_of<T, E, TERMS>(kr[u], kt);
      terms_of<T, E, TERMS>(vr[u], vt);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        if (masked >> u & 1) kt[t] = vt[t] = shortx8{0, 0, 0, 0, 0, 0, 0, 0};
        *reinterpret_cast<shortx8*>(kp + t * kPlaneK + key * kRowK + dim) = kt[t];
        *reinterpret_cast<shortx8*>(vp + t * kPlaneV + key * kRowV + dim) = vt[t];
      }
    }
    if (BIAS && tid < kKeys) biases[buf][tid] = b2;
  };

  floatx16 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;  // l_run: this lane's half of the row's sum

  const int tiles = (item.keys + kKeys - 1) / kKeys;
  const bool wave_live = wq * 32 < item.rows;
  if (tiles > 0) load(0);
  for (int t = 0; t < tiles; ++t) {
    const int buf = BUFS == 2 ? t & 1 : 0;
    if (BUFS == 1 && t > 0) __syncthreads();  // the tile before has been read
    store(buf);
    __syncthreads();
    if (t + 1 < tiles) load((t + 1) * kKeys);
    const int first = wk * KB * 32;  // this wave's states of the tile
    if (!wave_live || t * kKeys + first >= item.keys) continue;
    const short* kp = lds + buf * kBuffer + (first + l32) * kRowK + 8 * half;
    const short* vp = lds + buf * kBuffer + TERMS * kPlaneK + (first + 4 * half + (lane & 15) / 4) * kRowV +
                      (lane >> 4 & 1) * 16 + (lane & 3) * 4;

    floatx16 s[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
      for (int c = 0; c < kSlices; ++c) {
        shortx8 kt[TERMS];
#pragma unroll
        for (int i = 0; i < TERMS; ++i)
          kt[i] = *reinterpret_cast<const shortx8*>(kp + i * kPlaneK + b * 32 * kRowK + 16 * c);
        s[b] = products<E, TERMS>(kt, q[c], s[b]);
      }
      if constexpr (BIAS) {
        const float* br = &biases[buf][first + b * 32 + 4 * half];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float add = br[r / 4 * 8 + r % 4];
          s[b][r] = add == -INFINITY ? add : fmaf(s[b][r], to_log2, add);
        }
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
    const float ref = BIAS ? top - kLift<E> : fmaf(top, to_log2, -kLift<E>);
    if (__any(ref > m_run + kSlack)) {
      const float m_new = fmaxf(m_run, ref);
      // (-inf where nothing has been seen: its sums are zero)
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
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(BIAS ? s[b][r] - m : fmaf(s[b][r], to_log2, -m));
        sum[r & 3] += s[b][r];
      }
      l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[b][8 * c + i];
        shortx8 pt[TERMS];
        split8<E, TERMS>(x, pt);
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
          shortx8 vt[TERMS];
#pragma unroll
          for (int i = 0; i < TERMS; ++i) {
            const short* from = vp + i * kPlaneV + (b * 32 + 16 * c) * kRowV + 32 * d;
            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4*)(from));
            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) shortx4*)(from + 8 * kRowV));
            vt[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          }
          o[d] = products<E, TERMS>(vt, pt, o[d]);
        }
      }
    }
  }

  float l = l_run + other_half(l_run);
  if constexpr (WK > 1) {
    float* merge = reinterpret_cast<float*>(lds);
    constexpr int kWave = (DP / 2 + 2) * 64;
    __syncthreads();
    if (wk > 0) {
      float* mine = merge + ((wk - 1) * WQ + wq) * kWave;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[(b * 16 + r) * 64 + lane] = o[b][r];
      mine[DP / 2 * 64 + lane] = m_run;
      mine[(DP / 2 + 1) * 64 + lane] = l;
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int w = 0; w < WK - 1; ++w) {
      const float* theirs = merge + (w * WQ + wq) * kWave;
      const float m2 = theirs[DP / 2 * 64 + lane], l2 = theirs[(DP / 2 + 1) * 64 + lane];
      const float m_new = fmaxf(m_run, m2);
      const float keep = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      const float take = m2 == m_new ? 1.0f : __builtin_amdgcn_exp2f(m2 - m_new);
      m_run = m_new;
      l = l * keep + l2 * take;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] = o[b][r] * keep + theirs[(b * 16 + r) * 64 + lane] * take;
    }
  }
  if (!live) return;
  if (item.part >= 0) {
    constexpr int kRows = WQ * 32;
    float* part = p.partial + ((int64_t)item.part * p.kv_heads + kv) * (kRows * (DP + 2));
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<floatx4*>(part + row * DP + b * 32 + g * 8 + half * 4) =
            floatx4{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
    if (half == 0) {
      part[kRows * DP + row] = m_run;
      part[kRows * (DP + 1) + row] = l;
    }
    return;
  }
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;  // (nothing seen: zeros)
  T* out = static_cast<T*>(p.out) + token * p.out_token + head * p.out_head;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int dim = b * 32 + g * 8 + half * 4;
      T y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (T)(o[b][4 * g + e] * scale);
      if (vec) {
        if (dim < D) __builtin_memcpy(__builtin_assume_aligned(out + dim, 4 * sizeof(T)), y, sizeof(y));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dim + e < D) out[dim + e] = y[e];
      }
    }
}

template <class T, int TERMS, int DP, bool FEW>
int launch_tile(const CrossParams& p, hipStream_t stream) {
  constexpr CrossTile kTile = cross_tile(DP, TERMS, FEW);
  const int grid = p.item_count * p.kv_heads;
  if (p.bias)
    cross_kernel<T, TERMS, DP, FEW, true><<<grid, kTile.wq * kTile.wk * 64, 0, stream>>>(p);
  else
    cross_kernel<T, TERMS, DP, FEW, false><<<grid, kTile.wq * kTile.wk * 64, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <class T, int TERMS>
int launch_terms(const CrossParams& p, hipStream_t stream) {
  switch (cross_padded_dim(p.dim)) {
    case 64: return p.few ? launch_tile<T, TERMS, 64, true>(p, stream) : launch_tile<T, TERMS, 64, false>(p, stream);
    case 96: return p.few ? launch_tile<T, TERMS, 96, true>(p, stream) : launch_tile<T, TERMS, 96, false>(p, stream);
    default: return p.few ? launch_tile<T, TERMS, 128, true>(p, stream) : launch_tile<T, TERMS, 128, false>(p, stream);
  }
}

}  // namespace cross
}  // namespace tsplat
