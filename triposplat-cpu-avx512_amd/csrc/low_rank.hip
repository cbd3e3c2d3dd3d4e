// Low-rank adapters of many requests beside a shared Linear:
//   out[m] = y[m] + scale[a] (x[m] down[a]^T) up[a]^T,  a = rows[m].
//
// Two kernels: the inner values t = scale[a] x down[a]^T [M, R] go to scratch (R / K of x's bytes), the second joins
// t up[a]^T to y.  Both run on the bf16 matrix cores at fp32 precision: an fp32 value is the sum of three bf16 values
// (8 + 8 + 8 bits, split by truncation, so exactly and without overflow), a bf16 weight one, an fp16 weight two, an
// fp32 weight three; the products below 2^-23 of the whole are left out.
//
// Rows name their adapters in any order.  A workgroup handles a tile of rows and goes through the distinct adapters
// that its rows name; the matrix products run over the whole row tile, and only the rows of that adapter are written,
// so nothing that another row or another adapter holds (NaN, infinities) reaches a row.

#include <algorithm>
#include <type_traits>

#include "tsplat_common.h"
#include "tsplat_launch.h"

namespace tsplat {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// rows of x, y and out start at any float
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

union Pack8 {
  uint32_t w[4];
  bf16x8 v;
};

// The upper halves of a and b as two bf16 values.
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// v = sum of N bf16 values, each the truncation of what the ones before leave; exact for N = 3 (24 bits), and for
// N = 2 where v has 16 bits at most.  An infinity leaves NaN.
template <int N>
__device__ __forceinline__ void split(const float (&v)[8], bf16x8* out) {
  float left[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) left[i] = v[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    Pack8 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p.w[i] = upper_halves(left[2 * i], left[2 * i + 1]);
    out[n] = p.v;
    if (n + 1 < N) {
#pragma unroll
      for (int i = 0; i < 8; ++i) left[i] -= __uint_as_float(__float_as_uint(left[i]) & 0xffff0000u);
    }
  }
}

// An adapter's tile of 16 x 32 values: what a lane loads of it, and its bf16 terms.
template <int DTYPE>
struct Weights;

template <>
struct Weights<kAdapterBf16> {
  static constexpr int kTerms = 1, kBytes = 2;
  bf16x8 raw;
  __device__ __forceinline__ void load(const char* p) { raw = *reinterpret_cast<const bf16x8*>(p); }
  __device__ __forceinline__ void clear() { raw = bf16x8{}; }
  __device__ __forceinline__ void terms(bf16x8* t) const { t[0] = raw; }
};

template <>
struct Weights<kAdapterF16> {
  static constexpr int kTerms = 2, kBytes = 2;
  f16x8 raw;
  __device__ __forceinline__ void load(const char* p) { raw = *reinterpret_cast<const f16x8*>(p); }
  __device__ __forceinline__ void clear() { raw = f16x8{}; }
  __device__ __forceinline__ void terms(bf16x8* t) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
    split<2>(v, t);
  }
};

template <>
struct Weights<kAdapterF32> {
  static constexpr int kTerms = 3, kBytes = 4;
  floatx4 raw[2];
  __device__ __forceinline__ void load(const char* p) {
    raw[0] = reinterpret_cast<const floatx4*>(p)[0];
    raw[1] = reinterpret_cast<const floatx4*>(p)[1];
  }
  __device__ __forceinline__ void clear() { raw[0] = raw[1] = floatx4{}; }
  __device__ __forceinline__ void terms(bf16x8* t) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw[i >> 2][i & 3];
    split<3>(v, t);
  }
};

// The products of an fp32 value's terms with a weight's that count: i + j <= 2 (the others are below 2^-23 of the
// product), least first.
template <int TERMS>
constexpr int kProducts = TERMS == 1 ? 3 : TERMS == 2 ? 5 : 6;
template <int TERMS>
__device__ __forceinline__ constexpr int value_term(int i) {
  constexpr int one[] = {2, 1, 0}, two[] = {2, 1, 1, 0, 0}, three[] = {2, 1, 0, 1, 0, 0};
  return TERMS == 1 ? one[i] : TERMS == 2 ? two[i] : three[i];
}
template <int TERMS>
__device__ __forceinline__ constexpr int weight_term(int i) {
  constexpr int one[] = {0, 0, 0}, two[] = {0, 1, 0, 1, 0}, three[] = {0, 1, 2, 0, 1, 0};
  return TERMS == 1 ? one[i] : TERMS == 2 ? two[i] : three[i];
}

// Lane l (q = l / 16): weights row l % 16, inner index 8 q ..; values row l % 16 likewise; result rows 4 q + r of the
// weights, column l % 16 of the values.
__device__ __forceinline__ floatx4 mfma16(const bf16x8& w, const bf16x8& v, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, v, c, 0, 0, 0);
}

// The adapter of row m and its rank; id -1 for none.
__device__ __forceinline__ int row_adapter(const LowRankParams& p, int64_t m, bool live) {
  int id = live && m < p.M ? p.rows[m] : -1;
  if (id < 0 || id >= p.slots) return -1;
  return p.rank[id] > 0 ? id : -1;
}

// Goes through the distinct adapters of a tile of at most 64 rows (lane l holds row l's): f(adapter, mask of its
// rows).  With several passes (gridDim.z), every workgroup takes its share of them.
template <typename F>
__device__ __forceinline__ void each_adapter(int id, F f) {
  uint64_t left = __ballot(id >= 0);
  int pass = 0;
  while (left != 0) {
    const int a = __builtin_amdgcn_readlane(id, __ffsll((unsigned long long)left) - 1);
    const uint64_t mask = __ballot(id == a);
    left &= ~mask;
    if (pass % (int)gridDim.z == (int)blockIdx.z) f(a, mask);
    ++pass;
  }
}

// ------------------------------------------------------------------ t = scale x down^T
// A workgroup: RT * 16 rows x up to RB * 16 ranks; its W waves share the K axis in steps of 32 (neighbouring waves at
// neighbouring steps) and add their sums in LDS.  x goes from HBM to the registers that feed the matrix cores, each
// value read once by a wave; an adapter's tile of 16 ranks by 32 values is one contiguous load.
template <int DTYPE, int RT, int RB, int W>
__global__ __launch_bounds__(W * 64) void low_rank_down_kernel(LowRankParams p, int rank_blocks, int splits) {
  using Wt = Weights<DTYPE>;
  __shared__ floatx4 sums[W][W][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (RT * 16);
  const int rb0 = (int)(blockIdx.y % rank_blocks) * RB, part = (int)(blockIdx.y / rank_blocks);
  const int k_tiles = ceil_div(p.K, 32), r_tiles = ceil_div(p.R, 16), t_stride = r_tiles * 16;
  const int per_part = ceil_div(k_tiles, splits);
  const int s_end = min(k_tiles, (part + 1) * per_part);
  const int id = row_adapter(p, row0 + lane, lane < RT * 16);
  const float* xrow[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t m = row0 + t * 16 + (lane & 15);
    xrow[t] = p.x + (m < p.M ? m : p.M - 1) * p.x_stride + q * 8;
  }
  each_adapter(id, [&](int a, uint64_t mask) {
    const int tiles = min(RB, ceil_div(min(p.rank[a], p.R), 16) - rb0);
    if (tiles <= 0) return;  // the same for the whole workgroup
    const char* down = static_cast<const char*>(p.down) +
                       (((int64_t)a * r_tiles + rb0) * k_tiles * 512 + lane * 8) * Wt::kBytes;
    const int64_t tile_bytes = (int64_t)k_tiles * 512 * Wt::kBytes;
    floatx4 acc[RT][RB] = {};
    float raw[RT][8];
    auto load_x = [&](int s) {
      const int k = s * 32;
      if (k + 32 <= p.K) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const floatx4u lo = *reinterpret_cast<const floatx4u*>(xrow[t] + k);
          const floatx4u hi = *reinterpret_cast<const floatx4u*>(xrow[t] + k + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) raw[t][i] = lo[i], raw[t][4 + i] = hi[i];
        }
      } else {  // the last step of a K that is no multiple of 32
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i) raw[t][i] = k + q * 8 + i < p.K ? xrow[t][k + i] : 0.0f;
      }
    };
    int s = part * per_part + wave;
    if (s < s_end) load_x(s);
    for (; s < s_end; s += W) {
      Wt w[RB];
#pragma unroll
      for (int j = 0; j < RB; ++j)
        if (j < tiles) w[j].load(down + j * tile_bytes + (int64_t)s * 512 * Wt::kBytes);
      bf16x8 xs[RT][3];
#pragma unroll
      for (int t = 0; t < RT; ++t) split<3>(raw[t], xs[t]);
      if (s + W < s_end) load_x(s + W);
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        if (j >= tiles) break;
        bf16x8 ws[Wt::kTerms];
        w[j].terms(ws);
#pragma unroll
        for (int i = 0; i < kProducts<Wt::kTerms>; ++i)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            acc[t][j] = mfma16(ws[weight_term<Wt::kTerms>(i)], xs[t][value_term<Wt::kTerms>(i)], acc[t][j]);
      }
    }
    // the waves' sums, W tiles at a time: wave w adds up tile w
    const float scale = p.scale[a];
    float* out = p.scratch + (int64_t)part * p.M * t_stride;
#pragma unroll
    for (int first = 0; first < RT * RB; first += W) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (first + i < RT * RB) sums[i][wave][lane] = acc[(first + i) % RT][(first + i) / RT];
      __syncthreads();
      const int mine = first + wave, t = mine % RT, j = mine / RT;
      if (mine < RT * RB && j < tiles && (mask >> (t * 16 + (lane & 15)) & 1)) {
        floatx4 sum = sums[wave][0][lane];
#pragma unroll
        for (int i = 1; i < W; ++i) sum += sums[wave][i][lane];
        *reinterpret_cast<floatx4*>(out + (row0 + t * 16 + (lane & 15)) * t_stride + (rb0 + j) * 16 + q * 4) =
            sum * scale;
      }
    }
  });
}

// ------------------------------------------------------------------ out = y + t up^T
// A wave: RT * 16 rows x NT * 16 columns; its y is asked for before the products and joined after them.  A lane holds
// four neighbouring columns of a row.
template <int DTYPE, int RT, int NT, int W>
__global__ __launch_bounds__(W * 64) void low_rank_up_kernel(LowRankParams p, int splits) {
  using Wt = Weights<DTYPE>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (RT * 16);
  const int tile0 = (int)(blockIdx.y * W + wave) * NT;
  const int n_tiles = ceil_div(p.N, 16), r_steps = ceil_div(p.R, 32), t_stride = ceil_div(p.R, 16) * 16;
  if (tile0 >= n_tiles) return;
  const int tiles = min(NT, n_tiles - tile0), n0 = tile0 * 16 + q * 4;
  const int id = row_adapter(p, row0 + lane, lane < RT * 16);
  auto load_y = [&](int t, int j) {
    const float* src = p.y + (row0 + t * 16 + (lane & 15)) * p.y_stride;
    const int n = n0 + j * 16;
    if (n + 4 <= p.N) return (floatx4)*reinterpret_cast<const floatx4u*>(src + n);
    floatx4 v = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) v[i] = src[n + i];
    return v;
  };
  auto store = [&](int t, int j, floatx4 v) {
    float* dst = p.out + (row0 + t * 16 + (lane & 15)) * p.out_stride;
    const int n = n0 + j * 16;
    if (n + 4 <= p.N) {
      *reinterpret_cast<floatx4u*>(dst + n) = v;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) dst[n + i] = v[i];
  };
  each_adapter(id, [&](int a, uint64_t mask) {
    const int rank = min(p.rank[a], p.R), t_rank = ceil_div(rank, 16) * 16;
    floatx4 yv[RT][NT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
      if (mask >> (t * 16 + (lane & 15)) & 1) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (j < tiles) yv[t][j] = load_y(t, j);
      }
    floatx4 acc[RT][NT] = {};
    const char* up = static_cast<const char*>(p.up) +
                     (((int64_t)a * n_tiles + tile0) * r_steps * 512 + lane * 8) * Wt::kBytes;
    for (int s = 0; s * 32 < rank; ++s) {
      const int k = s * 32 + q * 8;
      Wt w[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        w[j].clear();
        if (j < tiles && k < rank) w[j].load(up + ((int64_t)j * r_steps + s) * 512 * Wt::kBytes);
      }
      bf16x8 ts[RT][3];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float v[8] = {};
        if (k < t_rank && (mask >> (t * 16 + (lane & 15)) & 1)) {
          const float* src = p.scratch + (row0 + t * 16 + (lane & 15)) * t_stride + k;
          for (int i = 0; i < splits; ++i, src += (int64_t)p.M * t_stride)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += src[e];
        }
        split<3>(v, ts[t]);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bf16x8 ws[Wt::kTerms];
        w[j].terms(ws);
#pragma unroll
        for (int i = 0; i < kProducts<Wt::kTerms>; ++i)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            acc[t][j] = mfma16(ws[weight_term<Wt::kTerms>(i)], ts[t][value_term<Wt::kTerms>(i)], acc[t][j]);
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
      if (mask >> (t * 16 + (lane & 15)) & 1) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (j < tiles) store(t, j, yv[t][j] + acc[t][j]);
      }
  });
  if (p.out == p.y || blockIdx.z != 0) return;
  const uint64_t bare = __ballot(id < 0);  // rows without an adapter
#pragma unroll
  for (int t = 0; t < RT; ++t)
    if ((bare >> (t * 16 + (lane & 15)) & 1) && row0 + t * 16 + (lane & 15) < p.M) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (j < tiles) store(t, j, load_y(t, j));
    }
}

// Rows a workgroup of the first kernel, the parts that it splits K into and the workgroups that share a row tile's
// adapters.  Few rows leave the chip idle without the last two.
struct Plan {
  int row_tiles, splits, passes;
};
constexpr int kDownWaves = 8;

Plan plan_of(int M, int K, int slots) {
  Plan pl{M > 8192 ? 4 : M > 4096 ? 2 : 1, 1, 1};
  const int wgs = ceil_div(M, 16 * pl.row_tiles);
  if (pl.row_tiles == 1) {
    pl.splits = std::max(1, std::min({256 / wgs, ceil_div(K, 32) / (2 * kDownWaves), 8}));
    pl.passes = std::max(1, std::min({1024 / wgs, 16, M, slots}));
  }
  return pl;
}

template <int DTYPE, int RT>
void launch_down(const LowRankParams& p, const Plan& pl, hipStream_t stream) {
  const int tiles = ceil_div(p.R, 16), m_blocks = ceil_div(p.M, 16 * RT);
  auto run = [&](auto rb) {
    constexpr int RB = decltype(rb)::value;
    const int blocks = ceil_div(tiles, RB);
    low_rank_down_kernel<DTYPE, RT, RB, kDownWaves>
        <<<dim3(m_blocks, blocks * pl.splits, pl.passes), kDownWaves * 64, 0, stream>>>(p, blocks, pl.splits);
  };
  if (tiles == 1)
    run(std::integral_constant<int, 1>{});
  else if (tiles == 2)
    run(std::integral_constant<int, 2>{});
  else
    run(std::integral_constant<int, 4>{});
}

template <int DTYPE>
void launch_typed(const LowRankParams& p, const Plan& pl, hipStream_t stream) {
  switch (pl.row_tiles) {
    case 1: launch_down<DTYPE, 1>(p, pl, stream); break;
    case 2: launch_down<DTYPE, 2>(p, pl, stream); break;
    default: launch_down<DTYPE, 4>(p, pl, stream); break;
  }
  constexpr int W = 4;
  const int n_tiles = ceil_div(p.N, 16);
  if (pl.row_tiles == 1) {
    low_rank_up_kernel<DTYPE, 1, 1, W>
        <<<dim3(ceil_div(p.M, 16), ceil_div(n_tiles, W), pl.passes), W * 64, 0, stream>>>(p, pl.splits);
  } else {
    low_rank_up_kernel<DTYPE, 2, 4, W>
        <<<dim3(ceil_div(p.M, 32), ceil_div(n_tiles, 4 * W), 1), W * 64, 0, stream>>>(p, pl.splits);
  }
}

}  // namespace

int64_t low_rank_scratch_bytes(int M, int K, int, int slots, int R, int) {
  return (int64_t)plan_of(M, K, slots).splits * M * ceil_div(R, 16) * 64;
}

int launch_low_rank_add(const LowRankParams& p, hipStream_t stream) {
  const Plan pl = plan_of(p.M, p.K, p.slots);
  switch (p.dtype) {
    case kAdapterF32: launch_typed<kAdapterF32>(p, pl, stream); break;
    case kAdapterBf16: launch_typed<kAdapterBf16>(p, pl, stream); break;
    default: launch_typed<kAdapterF16>(p, pl, stream); break;
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
