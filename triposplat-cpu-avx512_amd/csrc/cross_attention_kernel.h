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
// What bounds it, and measured: many rows, the exponents and what surrounds them in the vector units (a block of 32 x 32
// takes 125 vector instructions, 16 of them exponents at a quarter of the rate, and 8 products of 64 values a head): 275
// GFLOP of 2 x 16384 x 2048 in bf16 at 0.73 PFLOP/s, 375 us, 0.82 at 128 values a head.  Five ragged requests with a bias
// in bf16 92 us, 0.44 PFLOP/s: 784 workgroups of 22 and 32 tiles on 768 places (more parts than the plan makes cost more
// than they even out: 123).  fp32 values in three bf16 terms 1300 us for the former, 1.27 PFLOP/s of bf16 products, which is
// what a flagged call of cross_pairs.hip takes besides (unaligned 1570: loads of single values); in two terms 815, in one
// 425.  Few rows: HBM, 64 single tokens over 1.09 GB of bf16 states 221 us, 4.9 TB/s (a copy: 5.0); two single tokens over
// 50 MB of fp32 ones 22, of which about 5 join the parts and 6 are a launch and first loads.
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
// largest is still held (many small ones add up; sums of fp16 values are far from fp32's range).  bf16 has fp32's range, and
// so may its values: weights of 1 at most, 2^-kSlack where m has just moved, keep every sum that fp32 holds within it.  fp32
// values: a slack of 2, as x - m is rounded at its own size (8 rows over 30 states are off by 1.7e-7, with a slack of 8 by
// 2.4e-7; a normal row's largest score rises by less than that after its first tile).
template <class T>
constexpr float kSlack = sizeof(T) == 4 ? 2.0f : 8.0f;
template <class T>
constexpr float kLift = std::is_same_v<T, half_t> ? 7.0f : -kSlack<T>;

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
constexpr float kBf16Top = 3.3895313892515355e38f;  // the largest
template <bool CAP>
__device__ __forceinline__ int bf16_pair(float a, float b, float& left_a, float& left_b) {
  const bf16x2 first = CAP ? bf16x2{(bf16_t)__builtin_amdgcn_fmed3f(a, -kBf16Top, kBf16Top),
                                    (bf16_t)__builtin_amdgcn_fmed3f(b, -kBf16Top, kBf16Top)}
                           : bf16x2{(bf16_t)a, (bf16_t)b};
  const int w = __builtin_bit_cast(int, first);
  left_a = a - __int_as_float(w << 16);
  left_b = b - __int_as_float(w & 0xffff0000);
  return w;
}

// Eight values as TERMS vectors of 16-bit terms; CAP: the first terms within bf16's range.
template <class E, int TERMS, bool CAP = false>
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
        w[i] = t == 0 ? bf16_pair<CAP>(left[2 * i], left[2 * i + 1], a, b)
                      : bf16_pair<false>(left[2 * i], left[2 * i + 1], a, b);
        left[2 * i] = a, left[2 * i + 1] = b;
      }
      out[t] = __builtin_bit_cast(shortx8, w);
    }
  }
}

// Eight values of a row of D from dim on, as they are in memory (VEC: CrossParams::vec); past the row's end some others,
// which past_end makes zero: nothing waits for a load before its values are used.
template <class T>
struct Raw {
  T x[8];
};
template <class T, bool VEC>
__device__ __forceinline__ Raw<T> load_eight(const T* row, int dim, int D) {
  Raw<T> r;
  if constexpr (VEC) {
    __builtin_memcpy(&r, __builtin_assume_aligned(row + min(dim, D - 8), 16), sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = row[min(dim + i, D - 1)];
  }
  return r;
}
template <class T, bool VEC>
__device__ __forceinline__ Raw<T> past_end(Raw<T> r, int dim, int D, bool none) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (none || dim + (VEC ? 0 : i) >= D) r.x[i] = (T)0.0f;
  return r;
}

// The terms of eight values; of T's own 16 bits as they are.  A first term is bf16's largest at most, so that a finite value
// past it keeps finite terms (an infinity or NaN remains in the second).  A term alone rounds as bf16 does.
template <class T, class E, int TERMS>
__device__ __forceinline__ void terms_of(const Raw<T>& r, shortx8 (&out)[TERMS]) {
  if constexpr (sizeof(T) == 2) {
    out[0] = __builtin_bit_cast(shortx8, r);
  } else {
    split8<E, TERMS, (TERMS > 1)>(r.x, out);
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

// The second product's operand: eight states (four, and the four that lie 8 rows on) of a lane's column.
__device__ __forceinline__ shortx8 transposed(const short* from, int pitch) {
  const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)(from));
  const shortx4 hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)(from + 8 * pitch));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Keeps what follows behind what came before, where the compiler's order would need more registers than there are.
template <bool NOW>
__device__ __forceinline__ void in_order() {
  if constexpr (NOW) __builtin_amdgcn_sched_barrier(0);
}

// A workgroup's number among the grid's, such that neighbours are on one XCD.
__device__ __forceinline__ int xcd_order() {
  const int count = gridDim.x, per = count / 8, more = count % 8, xcd = blockIdx.x % 8;
  return xcd * per + min(xcd, more) + blockIdx.x / 8;
}

// Many rows: which item and key head a workgroup takes.  An XCD takes all tiles of the same key heads, which share their
// states in its L2, the longest first.
struct Work {
  int item, kv;
};
__device__ __forceinline__ Work work_of(const CrossParams& p) {
  if (p.kv_heads % 8 != 0) {
    const int id = xcd_order();
    return {id % p.item_count, id / p.item_count};
  }
  const int id = blockIdx.x / 8, heads = p.kv_heads / 8;
  return {id / heads, (int)(blockIdx.x % 8) * heads + id % heads};
}

// The query row of a lane: where q's vector and the result's lie.
struct Row {
  int64_t token;
  int head;
};
__device__ __forceinline__ Row row_of(const CrossParams& p, const CrossItem& item, int kv, int row) {
  const int at = item.row0 + row;
  return {item.token0 + at / p.group, kv * p.group + at % p.group};
}

// The thread's number again: what is made of it after a loop is not held in registers meanwhile.
__device__ __forceinline__ int thread_again() {
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  return tid;
}

// Columns 16 c + 8 half + i of a lane's query row in slice c; whether an infinity or NaN may be
// among them.
template <class T, class E, int TERMS, bool VEC, int SLICES>
__device__ __forceinline__ bool load_queries(const CrossParams& p, const Row& at, int half, shortx8 (&q)[SLICES][TERMS]) {
  const T* row = static_cast<const T*>(p.q) + at.token * p.q_token + at.head * p.q_head;
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < SLICES; ++c) {
    Raw<T> r = past_end<T, VEC>(load_eight<T, VEC>(row, 16 * c + 8 * half, p.dim), 16 * c + 8 * half, p.dim, false);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += fabsf((float)r.x[i]);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.x[i] *= p.scale * kLog2e;
    }
    terms_of<T, E, TERMS>(r, q[c]);
  }
  return !(sum < INFINITY);
}

// A bias in log2 units; a finite one stays finite (the type's lowest masks against others, not by itself; its largest leaves
// its own state alone).
__device__ __forceinline__ float bias_log2(float b) {
  constexpr float kTop = 3.4028234663852886e38f;
  return fabsf(b) < INFINITY ? __builtin_amdgcn_fmed3f(b * kLog2e, -kTop, kTop) : b;
}

// A product brought to T: rounded to fp32 first, whichever instructions the compiler would fuse it into.
template <class T>
__device__ __forceinline__ T rounded(float y) {
  asm("" : "+v"(y));
  return (T)y;
}

// What a block's sums become: a part, or the result.  The lane's row, 16 columns of each 32 in registers.
template <class T, int DP, bool VEC, int BLOCKS>
__device__ __forceinline__ void finish(const CrossParams& p, const CrossItem& item, int kv, int row, int tile_rows,
                                       const Row& at, int half, const floatx16 (&o)[BLOCKS], float m, float l) {
  if (item.part >= 0) {
    float* part = p.partial + ((int64_t)item.part * p.kv_heads + kv) * (tile_rows * (DP + 2));
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<floatx4*>(part + row * DP + b * 32 + g * 8 + half * 4) =
            floatx4{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
    if (half == 0) {
      part[tile_rows * DP + row] = m;
      part[tile_rows * (DP + 1) + row] = l;
    }
    return;
  }
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;  // (nothing seen: zeros)
  T* out = static_cast<T*>(p.out) + at.token * p.out_token + at.head * p.out_head;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int dim = b * 32 + g * 8 + half * 4;
      T y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = rounded<T>(o[b][4 * g + e] * scale);
      if (VEC) {
        if (dim < p.dim) __builtin_memcpy(__builtin_assume_aligned(out + dim, 4 * sizeof(T)), y, sizeof(y));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dim + e < p.dim) out[dim + e] = y[e];
      }
    }
}

// The weights of a block's 16 scores in log2 units and their sum; m the reference.
template <bool SCALED>
__device__ __forceinline__ float weights(floatx16& s, float to_log2, float m) {
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = __builtin_amdgcn_exp2f(SCALED ? s[r] - m : fmaf(s[r], to_log2, -m));
    sum[r & 3] += s[r];
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Many rows: a tile of states serves all of a workgroup's waves.
template <class T, int TERMS, int DP, bool BIAS, bool VEC>
__global__ __launch_bounds__(cross_tile(DP, TERMS, false).wq * 64, !VEC && DP > 64 && TERMS == 1 ? 1 : 2) void cross_kernel(
    CrossParams p) {
  typedef typename Element<T>::type E;
  constexpr CrossTile kTile = cross_tile(DP, TERMS, false);
  constexpr int KB = kTile.kb, kThreads = kTile.wq * 64, kKeys = KB * 32, kBlocks = DP / 32, kSlices = DP / 16;
  constexpr int kAllUnits = kKeys * DP / 8, kUnits = (kAllUnits + kThreads - 1) / kThreads;  // of 8 values
  constexpr int kRowK = DP + 8, kRowV = DP + 16;  // values from row to row
  constexpr bool kTight = DP > 96 && sizeof(T) == 4 && (TERMS == 1 || !VEC);
  constexpr int kPlaneK = kKeys * kRowK, kPlaneV = kKeys * kRowV;
  constexpr int kBuffer = TERMS * (kPlaneK + kPlaneV);
  __shared__ __attribute__((aligned(16))) short lds[2 * kBuffer];
  __shared__ __attribute__((aligned(16))) float biases[2][kKeys];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const Work work = work_of(p);
  if (p.flags && p.flags[(int64_t)work.item * p.kv_heads + work.kv] == 0) return;  // (done by the pairs)
  const CrossItem item = p.items[work.item];
  const int kv = work.kv, D = p.dim;

  // this lane's row
  const int row = wave * 32 + l32;
  const Row place = row_of(p, item, kv, row < item.rows ? row : 0);
  shortx8 q[kSlices][TERMS];
  const bool odd = __any(load_queries<T, E, TERMS, VEC>(p, place, half, q));
  const float to_log2 = sizeof(T) == 4 ? 1.0f : p.scale * kLog2e;

  const T* kbase = static_cast<const T*>(p.k) + (int64_t)item.key0 * p.k_token + kv * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + (int64_t)item.key0 * p.v_token + kv * p.v_head;
  const float* bias = p.bias ? p.bias + item.key0 : nullptr;
  auto bias_of = [&](int64_t key) { return VEC || bias ? bias[key] : 0.0f; };  // (unaligned calls: with or without one)

  Raw<T> kr[kUnits], vr[kUnits];
  float br[kUnits], b2 = 0.0f;  // the biases of the units' states, of state key0 + tid
  auto load = [&](int key0) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, dim = unit % (DP / 8) * 8;
      const int64_t from = min(key0 + unit / (DP / 8), item.keys - 1);
      kr[u] = load_eight<T, VEC>(kbase + from * p.k_token, dim, D);
      in_order<kTight>();
      vr[u] = load_eight<T, VEC>(vbase + from * p.v_token, dim, D);
      if (BIAS) br[u] = bias_of(from);
      in_order<kTight>();
    }
    if (BIAS && tid < kKeys) b2 = bias_of(min(key0 + tid, item.keys - 1));
  };
  auto store = [&](int key0, int buf) {
    short* kp = lds + buf * kBuffer;
    short* vp = kp + TERMS * kPlaneK;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = tid + u * kThreads, key = unit / (DP / 8), dim = unit % (DP / 8) * 8;
      if (kAllUnits % kThreads && unit >= kAllUnits) break;
      const bool none = key0 + key >= item.keys || (BIAS && br[u] == -INFINITY);
      shortx8 kt[TERMS], vt[TERMS];
      terms_of<T, E, TERMS>(past_end<T, VEC>(kr[u], dim, D, none), kt);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) *reinterpret_cast<shortx8*>(kp + t * kPlaneK + key * kRowK + dim) = kt[t];
      in_order<kTight>();
      terms_of<T, E, TERMS>(past_end<T, VEC>(vr[u], dim, D, none), vt);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) *reinterpret_cast<shortx8*>(vp + t * kPlaneV + key * kRowV + dim) = vt[t];
    }
    if (BIAS && tid < kKeys) biases[buf][tid] = key0 + tid < item.keys ? bias_log2(b2) : -INFINITY;
  };

  floatx16 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;  // l_run: this lane's half of the row's sum

  const int tiles = (item.keys + kKeys - 1) / kKeys;
  const bool wave_live = wave * 32 < item.rows;
  constexpr bool kLate = DP > 96 && TERMS == 3 && !VEC;  // (no registers to hold a tile while another is multiplied)
  if (!kLate && tiles > 0) load(0);
  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1;
    if (kLate) load(t * kKeys);
    store(t * kKeys, buf);
    __syncthreads();
    if (!kLate && t + 1 < tiles) load((t + 1) * kKeys);
    if (!wave_live) continue;
    const short* kp = lds + buf * kBuffer + l32 * kRowK + 8 * half;
    const short* vp = lds + buf * kBuffer + TERMS * kPlaneK + (4 * half + (lane & 15) / 4) * kRowV +
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
        in_order<kTight>();
      }
      if constexpr (BIAS) {
        const float* br = &biases[buf][b * 32 + 4 * half];
        if (odd) {  // (a masked state's zeros times an infinity)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (br[r / 4 * 8 + r % 4] == -INFINITY) s[b][r] = 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = fmaf(s[b][r], to_log2, br[r / 4 * 8 + r % 4]);
      } else {
        const int left = item.keys - (t * kKeys + b * 32) - 4 * half;  // states of this block from this lane's first
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
    const float ref = BIAS ? top - kLift<T> : fmaf(top, to_log2, -kLift<T>);
    if (__any(ref > m_run + kSlack<T>)) {
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
      l_run += weights<BIAS>(s[b], to_log2, m);
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
          for (int i = 0; i < TERMS; ++i)
            vt[i] = transposed(vp + i * kPlaneV + (b * 32 + 16 * c) * kRowV + 32 * d, kRowV);
          o[d] = products<E, TERMS>(vt, pt, o[d]);
          in_order<kTight>();
        }
      }
    }
  }

  const float l = l_run + other_half(l_run);
  const int again = thread_again(), out_row = (again >> 6) * 32 + (again & 31);
  if (out_row < item.rows)
    finish<T, DP, VEC>(p, item, kv, out_row, kTile.wq * 32, row_of(p, item, kv, out_row), again >> 5 & 1, o, m_run, l);
}

// At most 32 rows a request, where reading the states is all: each wave takes every fourth block of 32 states by itself,
// without a barrier, K and V through the wave's own LDS; the next block's loads are under way while this
// one is multiplied.  The waves'
// sums meet at the end.
template <class T, int TERMS, int DP, bool BIAS, bool VEC>
__global__ __launch_bounds__(kFewWaves * 64, DP > 64 && (sizeof(T) == 4 || !VEC) ? 1 : 2) void cross_few_kernel(CrossParams p) {
  typedef typename Element<T>::type E;
  constexpr int kBlocks = DP / 32, kSlices = DP / 16, kUnits = DP / 16;  // a lane's eights of 32 states' values
  constexpr int kRowK = DP + 8, kRowV = DP + 16;
  constexpr bool kTight = DP > 96;
  constexpr int kMerge = (kFewWaves - 1) * (DP / 2 + 2) * 64 * 2;  // shorts of the sums that meet
  constexpr int kPlane = 32 * kRowV, kRows = kFewWaves * TERMS * kPlane;  // (K's rows fit as well)
  constexpr int kLds = kRows > kMerge ? kRows : kMerge;
  __shared__ __attribute__((aligned(16))) short lds[kLds];
  __shared__ __attribute__((aligned(16))) float biases[kFewWaves][32];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  // (an item's key heads are neighbours: their states lie side by side in memory)
  const int id = xcd_order();
  const CrossItem item = p.items[id / p.kv_heads];
  const int kv = id % p.kv_heads;
  const int D = p.dim;
  const bool live = l32 < item.rows;
  const Row place = row_of(p, item, kv, live ? l32 : 0);
  const float to_log2 = sizeof(T) == 4 ? 1.0f : p.scale * kLog2e;

  const T* kbase = static_cast<const T*>(p.k) + (int64_t)item.key0 * p.k_token + kv * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + (int64_t)item.key0 * p.v_token + kv * p.v_head;
  const float* bias = p.bias ? p.bias + item.key0 : nullptr;
  short* wlds = lds + wave * TERMS * kPlane;
  Raw<T> kr[kUnits], vr[kUnits];
  float b2 = 0.0f;
  const int last = item.keys - 1;  // (past the last state: its values, which count for nothing)
  auto load_rows = [&](Raw<T>(&r)[kUnits], const T* base, int64_t step, int key0) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = lane + u * 64;
      r[u] = load_eight<T, VEC>(base + min(key0 + unit / (DP / 8), last) * step, unit % (DP / 8) * 8, D);
    }
  };
  auto load_k = [&](int key0) {
    load_rows(kr, kbase, p.k_token, key0);
    if (BIAS) b2 = VEC || bias ? bias[min(key0 + l32, last)] : 0.0f;
  };
  auto load_v = [&](int key0) { load_rows(vr, vbase, p.v_token, key0); };
  // Their terms to the wave's LDS, a plane of rows of `pitch` for each; zeros where nothing counts.  (A wave's LDS
  // operations are done in order.)
  auto put_rows = [&](const Raw<T>(&r)[kUnits], int pitch, int left) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = lane + u * 64, state = unit / (DP / 8), dim = unit % (DP / 8) * 8;
      const bool none = state >= left || (BIAS && biases[wave][state] == -INFINITY);
      shortx8 out[TERMS];
      terms_of<T, E, TERMS>(past_end<T, VEC>(r[u], dim, D, none), out);
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
        *reinterpret_cast<shortx8*>(wlds + t * kPlane + state * pitch + dim) = out[t];
    }
    __builtin_amdgcn_wave_barrier();
  };
  const short* kp = wlds + l32 * kRowK + 8 * half;
  const short* vp = wlds + (4 * half + (lane & 15) / 4) * kRowV + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
  const float* br = &biases[wave][4 * half];

  floatx16 o[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  constexpr int kStep = kFewWaves * 32;
  int key0 = wave * 32;
  if (key0 <= last) {
    load_k(key0);
    load_v(key0);
  }
  shortx8 q[kSlices][TERMS];
  load_queries<T, E, TERMS, VEC>(p, place, half, q);
  for (; key0 <= last; key0 += kStep) {
    const int left = item.keys - key0;  // states from this block's first on
    if (BIAS) {
      biases[wave][l32] = l32 < left ? bias_log2(b2) : -INFINITY;  // (both halves write the same)
      __builtin_amdgcn_wave_barrier();
    }
    const bool more = key0 + kStep <= last;
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
    put_rows(kr, kRowK, left);
    if (more) load_k(key0 + kStep);
#pragma unroll
    for (int c = 0; c < kSlices; ++c) {
      shortx8 kt[TERMS];
#pragma unroll
      for (int t = 0; t < TERMS; ++t) kt[t] = *reinterpret_cast<const shortx8*>(kp + t * kPlane + 16 * c);
      s = products<E, TERMS>(kt, q[c], s);
      in_order<kTight>();
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = r / 4 * 8 + r % 4;
      if constexpr (BIAS) {
        const float add = br[key];
        s[r] = add == -INFINITY ? add : fmaf(s[r], to_log2, add);
      } else {
        s[r] = key + 4 * half < left ? s[r] : -INFINITY;
      }
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaxf(top, other_half(top));
    const float ref = BIAS ? top - kLift<T> : fmaf(top, to_log2, -kLift<T>);
    if (__any(ref > m_run + kSlack<T>)) {
      const float m_new = fmaxf(m_run, ref);
      const float keep = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= keep;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] *= keep;
      m_run = m_new;
    }
    l_run += weights<BIAS>(s, to_log2, m_run == -INFINITY ? 0.0f : m_run);
    shortx8 pt[2][TERMS];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s[8 * c + i];
      split8<E, TERMS>(x, pt[c]);
    }
    put_rows(vr, kRowV, left);
    if (more) load_v(key0 + kStep);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) {
        shortx8 vt[TERMS];
#pragma unroll
        for (int t = 0; t < TERMS; ++t) vt[t] = transposed(vp + t * kPlane + 16 * c * kRowV + 32 * d, kRowV);
        o[d] = products<E, TERMS>(vt, pt[c], o[d]);
        in_order<kTight>();
      }
    __builtin_amdgcn_wave_barrier();
  }

  float l = l_run + other_half(l_run);
  float* merge = reinterpret_cast<float*>(lds);
  constexpr int kWave = (DP / 2 + 2) * 64;
  __syncthreads();
  if (wave > 0) {
    float* mine = merge + (wave - 1) * kWave;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(b * 16 + r) * 64 + lane] = o[b][r];
    mine[DP / 2 * 64 + lane] = m_run;
    mine[(DP / 2 + 1) * 64 + lane] = l;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 0; w < kFewWaves - 1; ++w) {
    const float* theirs = merge + w * kWave;
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
  if (live) finish<T, DP, VEC>(p, item, kv, l32, 32, place, half, o, m_run, l);
}

template <class T, int TERMS, int DP, bool BIAS, bool VEC>
int launch_kernel(const CrossParams& p, hipStream_t stream) {
  const int grid = p.item_count * p.kv_heads;
  if (p.few)
    cross_few_kernel<T, TERMS, DP, BIAS, VEC><<<grid, kFewWaves * 64, 0, stream>>>(p);
  else
    cross_kernel<T, TERMS, DP, BIAS, VEC><<<grid, cross_tile(DP, TERMS, false).wq * 64, 0, stream>>>(p);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <class T, int TERMS, int DP>
int launch_dim(const CrossParams& p, hipStream_t stream) {
  if (!p.vec) return launch_kernel<T, TERMS, DP, true, false>(p, stream);
  return p.bias ? launch_kernel<T, TERMS, DP, true, true>(p, stream) : launch_kernel<T, TERMS, DP, false, true>(p, stream);
}

template <class T, int TERMS>
int launch_terms(const CrossParams& p, hipStream_t stream) {
  switch (cross_padded_dim(p.dim)) {
    case 64: return launch_dim<T, TERMS, 64>(p, stream);
    case 96: return launch_dim<T, TERMS, 96>(p, stream);
    default: return launch_dim<T, TERMS, 128>(p, stream);
  }
}

}  // namespace cross
}  // namespace tsplat
