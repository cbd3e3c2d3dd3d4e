// Low-rank adapters of many requests beside a shared Linear:
//   out[m] = y[m] + scale[a] (x[m] down[a]^T) up[a]^T,  a = rows[m].
//
// Two kernels: the inner values t = scale[a] x down[a]^T [M, R] go to scratch (R / K of x's bytes), the second joins
// t up[a]^T to y.  Both run on the bf16 matrix cores at fp32 precision: an fp32 value is the sum of three bf16 values
// (8 + 8 + 8 bits, split by truncation, so exactly and without overflow), a bf16 weight one, an fp16 weight two, an
// fp32 weight three; the smallest products of terms are left out (kProducts says what that costs).
//
// What bounds it: 12294 x 1024 -> 4096, rank 16, HBM: 453 MB in 89-92 us (5.0 TB/s; x 18, y 74).  16384 x 4096 -> 1024,
// rank 64 in fp32 (402 MB, 79 us at a copy's rate): 136-142 us for one adapter, 152 where two requests meet.  The first
// kernel's waves wait for loads half of their time, two of them a SIMD for their 194 registers, while every 32 rows read
// the adapter's 1.5 MB through L2 (0.97 GB at 9 TB/s, two thirds of it hits), and the border tile's second adapter ends
// last.  Adapter values staged in LDS for 64 or 128 rows were slower or no faster: a barrier a step of K, and t in parts.
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
struct Weights<kAdapterF32> {  // three planes of the tile, split when the bank was laid out
  static constexpr int kTerms = 3, kBytes = 6;
  bf16x8 raw[3];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < 3; ++i) raw[i] = *reinterpret_cast<const bf16x8*>(p + i * 1024);
  }
  __device__ __forceinline__ void clear() { raw[0] = raw[1] = raw[2] = bf16x8{}; }
  __device__ __forceinline__ void terms(bf16x8* t) const {
#pragma unroll
    for (int i = 0; i < 3; ++i) t[i] = raw[i];
  }
};

// The products of an fp32 value's terms with a weight's that count: i + j <= 2, least first.  By truncation term 1 is
// below 2^-7 of its value and term 2 below 2^-15, so what is left out is below 2^-22 of the product for fp16 weights
// (2 with 1), below 2^-21 for fp32 ones (1 with 2, 2 with 1, 2 with 2), nothing for bf16.  All terms have their value's
// sign: it always takes from the product (0.7 x 2^-24 on average for fp32 weights; a sum's own roundings are more).
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

// Scratch: what the first kernel finds out about each row, its adapter and that one's rank in one number (-1: none),
// then its inner values [splits][M][ceil(R/16) 16].  With that the second kernel's loads hang on one load, not three,
// each of which takes microseconds while memory is saturated.
__host__ __device__ constexpr int64_t meta_floats(int M) { return ((int64_t)M + 63) / 64 * 64; }
constexpr int kIdBits = 20;
static_assert((1 << (31 - kIdBits)) > 512, "a rank of 512 has room above the adapter's number");

// Goes through the distinct adapters of a tile of at most 64 rows: lane l holds row l's number, negative for none;
// f(number, its first row, mask of its rows).  Of several passes, this workgroup's share of them.
template <typename F>
__device__ __forceinline__ void each_adapter(int number, uint64_t rows, int passes, F f) {
  uint64_t left = __ballot(number >= 0) & rows;
  int pass = 0;
  while (left != 0) {
    const int first = __ffsll((unsigned long long)left) - 1;
    const int a = __builtin_amdgcn_readlane(number, first);
    const uint64_t mask = __ballot(number == a) & rows;
    left &= ~mask;
    if (passes == 1 || pass % passes == (int)blockIdx.z) f(a, first, mask);
    ++pass;
  }
}

// ------------------------------------------------------------------ t = scale x down^T
// A workgroup: RT * 16 rows x up to RB * 16 ranks; its W waves share the K axis in runs of 32-value steps and add their
// sums in LDS.  x goes from HBM to the registers that feed the matrix cores, a step ahead, each value read once by one
// wave; an adapter's tile of 16 ranks by 32 values is one contiguous load, a step ahead too.  (Two or four steps of x
// ahead are 5-40 % slower: the loads of all waves fill memory's queues as it is.)
struct DownRange {
  int rb0, part, s_begin, s_end;  // first rank tile, part of K, the wave's steps
};

// RT row tiles from row0 through adapter a's `tiles` rank tiles; bit i of mask: row0 + i is the adapter's.
template <int DTYPE, int RT, int RB, int W>
struct DownTile {
  using Wt = Weights<DTYPE>;
  static constexpr int kRound = RT * RB < W ? RT * RB : W;  // tiles added up at once
  float raw[RT][8];

  __device__ __forceinline__ void load_x(const LowRankParams& p, int64_t row0, int s) {
    const int lane = threadIdx.x & 63, k = s * 32 + (lane >> 4) * 8;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int64_t m = row0 + t * 16 + (lane & 15);
      const float* src = p.x + (m < p.M ? m : p.M - 1) * p.x_stride + k;
      if (s * 32 + 32 <= p.K) {
        const floatx4u lo = *reinterpret_cast<const floatx4u*>(src);
        const floatx4u hi = *reinterpret_cast<const floatx4u*>(src + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[t][i] = lo[i], raw[t][4 + i] = hi[i];
      } else {  // the last step of a K that is no multiple of 32
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[t][i] = k + i < p.K ? src[i] : 0.0f;
      }
    }
  }

  // x of the first step is in raw; w holds the first step's weights.
  __device__ __forceinline__ void run(const LowRankParams& p, const DownRange& r, int64_t row0, Wt (&w)[RB],
                                      const char* down, int64_t tile_bytes, int tiles, float scale, uint64_t mask,
                                      floatx4 (*sums)[W][64]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
    const int t_stride = ceil_div(p.R, 16) * 16;
    floatx4 acc[RT][RB] = {};
    for (int s = r.s_begin; s < r.s_end; ++s) {
      bf16x8 xs[RT][3];
#pragma unroll
      for (int t = 0; t < RT; ++t) split<3>(raw[t], xs[t]);
      if (s + 1 < r.s_end) load_x(p, row0, s + 1);
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
        if (s + 1 < r.s_end) w[j].load(down + j * tile_bytes + (int64_t)(s + 1) * 512 * Wt::kBytes);
      }
    }
    // the waves' sums, kRound tiles at a time: wave i adds up tile i
    float* out = p.scratch + meta_floats(p.M) + (int64_t)r.part * p.M * t_stride;
#pragma unroll
    for (int at = 0; at < RT * RB; at += kRound) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRound; ++i)
        if (at + i < RT * RB) sums[i][wave][lane] = acc[(at + i) % RT][(at + i) / RT];
      __syncthreads();
      const int mine = at + wave, t = mine % RT, j = mine / RT;
      if (wave < kRound && mine < RT * RB && j < tiles && (mask >> (t * 16 + (lane & 15)) & 1)) {
        floatx4 sum = sums[wave][0][lane];
#pragma unroll
        for (int i = 1; i < W; ++i) sum += sums[wave][i][lane];
        *reinterpret_cast<floatx4*>(out + (row0 + t * 16 + (lane & 15)) * t_stride + (r.rb0 + j) * 16 + q * 4) =
            sum * scale;
      }
    }
  }
};

template <int DTYPE, int RT, int RB, int W>
__global__ __launch_bounds__(W * 64) void low_rank_down_kernel(LowRankParams p, int rank_blocks, int splits,
                                                               int passes) {
  using Wt = Weights<DTYPE>;
  __shared__ floatx4 sums[DownTile<DTYPE, RT, RB, W>::kRound][W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (int64_t)blockIdx.x * (RT * 16);
  const int k_tiles = ceil_div(p.K, 32), r_tiles = ceil_div(p.R, 16), share = ceil_div(k_tiles, splits * W);
  DownRange r;
  r.rb0 = (int)(blockIdx.y % rank_blocks) * RB;
  r.part = (int)(blockIdx.y / rank_blocks);
  r.s_begin = (r.part * W + wave) * share;
  r.s_end = min(k_tiles, r.s_begin + share);
  // x is on its way before its rows' adapters are known; a pass that may have none waits
  DownTile<DTYPE, RT, RB, W> all;
  bool held = RT == 1 ? blockIdx.z == 0 : (int)blockIdx.z == passes - 1;
  if (held && r.s_begin < r.s_end) all.load_x(p, row0, r.s_begin);
  int id = lane < RT * 16 && row0 + lane < p.M ? p.rows[row0 + lane] : -1;
  if (id >= p.slots) id = -1;
  const int row_rank = id >= 0 ? min(p.rank[id], p.R) : 0;
  auto adapter = [&](int a, int first_row, uint64_t mask) {
    const char* down = static_cast<const char*>(p.down) +
                       ((int64_t)a * r_tiles + r.rb0) * k_tiles * 512 * Wt::kBytes + lane * 16;
    const int64_t tile_bytes = (int64_t)k_tiles * 512 * Wt::kBytes;
    const float scale = p.scale[a];
    Wt w[RB];
    auto load_w = [&](int tiles) {
#pragma unroll
      for (int j = 0; j < RB; ++j)
        if (j < tiles && r.s_begin < r.s_end) w[j].load(down + j * tile_bytes + (int64_t)r.s_begin * 512 * Wt::kBytes);
    };
    load_w(min(RB, r_tiles - r.rb0));  // (of the bank: these do not wait for the adapter's own rank)
    const int rank = __builtin_amdgcn_readlane(row_rank, first_row);
    const int tiles = rank > 0 ? min(RB, ceil_div(rank, 16) - r.rb0) : 0;
    if (tiles <= 0) return;  // the same for the whole workgroup
    if (RT == 1 || held) {
      if (!held && r.s_begin < r.s_end) all.load_x(p, row0, r.s_begin);
      held = false;
      all.run(p, r, row0, w, down, tile_bytes, tiles, scale, mask, sums);
      return;
    }
    // A further adapter of a wider tile, at the border of two requests: its row tiles by themselves.
    bool again = false;
    for (int t = 0; t < RT; ++t) {
      const uint64_t rows = mask >> (t * 16) & 0xffff;
      if (rows == 0) continue;
      if (again) load_w(tiles);
      again = true;
      DownTile<DTYPE, 1, RB, W> one;
      if (r.s_begin < r.s_end) one.load_x(p, row0 + t * 16, r.s_begin);
      one.run(p, r, row0 + t * 16, w, down, tile_bytes, tiles, scale, rows, sums);
    }
  };
  if constexpr (RT == 1) {
    each_adapter(id, ~0ull, passes, adapter);
  } else {
    // The middle row's adapter has the most rows of a border tile: it goes through all row tiles at once.  The others,
    // where a pass of their own is asked for, go before: most of its workgroups end at once, and those of a border start
    // early, where one workgroup would take twice its time and end last.
    const int middle = __builtin_amdgcn_readlane(id, RT * 8);
    if (held && middle >= 0) adapter(middle, RT * 8, __ballot(id == middle));
    if (blockIdx.z == 0) each_adapter(id == middle ? -1 : id, ~0ull, 1, adapter);
  }
  if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0 && lane < RT * 16 && row0 + lane < p.M)
    reinterpret_cast<int*>(p.scratch)[row0 + lane] = row_rank > 0 ? row_rank << kIdBits | id : -1;
}

// ------------------------------------------------------------------ out = y + t up^T
// A wave: 16 rows x NT * 16 columns.  Its y, its rows' numbers and inner values are asked for at once, then the
// weights, 32 ranks at a time.  A lane holds four neighbouring columns of a row.  Workgroups follow one another along the
// rows, as the values lie in memory: that order alone is worth 15 % of the bandwidth.
template <int DTYPE, int NT, int W>
__global__ __launch_bounds__(W * 64) void low_rank_up_kernel(LowRankParams p, int splits, int passes) {
  using Wt = Weights<DTYPE>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
  const int64_t row0 = (blockIdx.y + (passes == 1 ? (int64_t)blockIdx.z * gridDim.y : 0)) * 16;
  const int tile0 = (int)(blockIdx.x * W + wave) * NT;
  const int n_tiles = ceil_div(p.N, 16), r_steps = ceil_div(p.R, 32), t_stride = ceil_div(p.R, 16) * 16;
  if (tile0 >= n_tiles || row0 >= p.M) return;
  const int64_t m = row0 + (lane & 15);
  const bool there = m < p.M;
  const float* yrow = p.y + m * p.y_stride + tile0 * 16 + q * 4;
  float* orow = p.out + m * p.out_stride + tile0 * 16 + q * 4;
  const float* trow = p.scratch + meta_floats(p.M) + m * t_stride + q * 8;
  const int left = p.N - tile0 * 16 - q * 4;  // columns from this lane's first
  auto run = [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;  // all NT tiles have all their columns
    floatx4 yv[NT];
    auto load_y = [&] {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (kWhole || left >= j * 16 + 4) {
          yv[j] = *reinterpret_cast<const floatx4u*>(yrow + j * 16);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (left > j * 16 + i) yv[j][i] = yrow[j * 16 + i];
        }
      }
    };
    auto store = [&](const floatx4 (&v)[NT]) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (kWhole || left >= j * 16 + 4) {
          *reinterpret_cast<floatx4u*>(orow + j * 16) = v[j];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (left > j * 16 + i) orow[j * 16 + i] = v[j][i];
        }
      }
    };
    float inner[8];  // past the adapter's rank: whatever scratch holds
    auto load_inner = [&](int k) {
      if (k + q * 8 >= t_stride) return;
      const float* src = trow + k;
#pragma unroll
      for (int e = 0; e < 8; ++e) inner[e] = src[e];
      for (int i = 1; i < splits; ++i) {
        src += (int64_t)p.M * t_stride;
#pragma unroll
        for (int e = 0; e < 8; ++e) inner[e] += src[e];
      }
    };
    int meta = -1;
    if (there) {
      meta = reinterpret_cast<const int*>(p.scratch)[m];
      load_inner(0);
      if (passes == 1) load_y();
    }
    bool held = true;
    each_adapter(meta, 0xffff, passes, [&](int number, int, uint64_t) {
      const int a = number & ((1 << kIdBits) - 1), rank = number >> kIdBits;
      const char* up = static_cast<const char*>(p.up) +
                       ((int64_t)a * n_tiles + tile0) * r_steps * 512 * Wt::kBytes + lane * 16;
      const bool mine = meta == number;
      const int t_rank = mine ? ceil_div(rank, 16) * 16 : 0;
      floatx4 acc[NT] = {};
      for (int k = 0; k < rank; k += 32, up += 512 * Wt::kBytes) {
        Wt w[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          w[j].clear();
          if (k + q * 8 < rank && (kWhole || tile0 + j < n_tiles)) w[j].load(up + (int64_t)j * r_steps * 512 * Wt::kBytes);
        }
        if (!held && there) load_inner(k);
        held = r_steps == 1;
        if (k == 0 && passes != 1 && mine) load_y();
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + q * 8 < t_rank ? inner[e] : 0.0f;
        bf16x8 ts[3];
        split<3>(v, ts);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          bf16x8 ws[Wt::kTerms];
          w[j].terms(ws);
#pragma unroll
          for (int i = 0; i < kProducts<Wt::kTerms>; ++i)
            acc[j] = mfma16(ws[weight_term<Wt::kTerms>(i)], ts[value_term<Wt::kTerms>(i)], acc[j]);
        }
      }
      if (mine) {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] += yv[j];
        store(acc);
      }
    });
    if (p.out == p.y || (passes != 1 && blockIdx.z != 0)) return;
    if (there && meta < 0) {  // rows without an adapter
      if (passes != 1) load_y();
      store(yv);
    }
  };
  if ((tile0 + NT) * 16 <= p.N)
    run(std::true_type{});
  else
    run(std::false_type{});
}

// ------------------------------------------------------------------ few rows: both products in one launch
// A workgroup: 16 rows x W NT * 16 columns, ranks up to 32.  Its waves share the K axis for the inner values of every
// row, add their sums in LDS, and each multiplies them with its own columns' weights.  Every column block computes the
// inner values anew, which costs less than a second launch and the wait between the two while that is little work:
// 2 rows, 1024 -> 1024, rank 16: 5.0 us against 7.0, and 4 us less of the host; see few_rows() for where it turns.
template <int DTYPE, int NT, int W>
__global__ __launch_bounds__(W * 64) void low_rank_few_kernel(LowRankParams p, int passes) {
  using Wt = Weights<DTYPE>;
  constexpr int kInner = 32 + 4;  // floats a row in LDS: 16-byte reads of neighbouring rows in other banks
  __shared__ floatx4 sums[2][W][64];
  __shared__ __attribute__((aligned(16))) float inner[16 * kInner];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.y * 16, m = row0 + (lane & 15);
  const int k_tiles = ceil_div(p.K, 32), r_tiles = ceil_div(p.R, 16);
  const int n_tiles = ceil_div(p.N, 16), tile0 = (int)(blockIdx.x * W + wave) * NT;
  const int share = ceil_div(k_tiles, W), s_begin = wave * share, s_end = min(k_tiles, s_begin + share);
  const float* xrow = p.x + (m < p.M ? m : p.M - 1) * p.x_stride + q * 8;
  const int n0 = tile0 * 16 + q * 4;
  int id = m < p.M ? p.rows[m] : -1;
  if (id >= p.slots) id = -1;
  const int row_rank = id >= 0 ? min(p.rank[id], p.R) : 0;
  floatx4 yv[NT];
  auto load_y = [&] {
    const float* src = p.y + m * p.y_stride;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + j * 16 + i < p.N) yv[j][i] = src[n0 + j * 16 + i];
  };
  auto store = [&](const floatx4 (&v)[NT]) {
    float* dst = p.out + m * p.out_stride;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + j * 16 + i < p.N) dst[n0 + j * 16 + i] = v[j][i];
  };
  each_adapter(id, 0xffff, passes, [&](int a, int first_row, uint64_t mask) {
    const int rank = __builtin_amdgcn_readlane(row_rank, first_row);
    if (rank <= 0) return;  // the same for the whole workgroup
    const bool mine = mask >> (lane & 15) & 1;
    const float scale = p.scale[a];
    if (mine) load_y();
    floatx4 acc[NT] = {};
    const int tiles = ceil_div(rank, 16);
    const char* down = static_cast<const char*>(p.down) + (int64_t)a * r_tiles * k_tiles * 512 * Wt::kBytes + lane * 16;
    const char* up = static_cast<const char*>(p.up) + ((int64_t)a * n_tiles + tile0) * 512 * Wt::kBytes + lane * 16;
    Wt wu[NT];  // the second product's weights come while the first runs
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      wu[j].clear();
      if (tile0 + j < n_tiles && q * 8 < rank) wu[j].load(up + j * 512 * Wt::kBytes);
    }
    floatx4 t[2] = {};
    for (int s = s_begin; s < s_end; ++s) {
      const int k = s * 32;
      Wt w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j < tiles) w[j].load(down + ((int64_t)j * k_tiles + s) * 512 * Wt::kBytes);
      float v[8];
      if (k + 32 <= p.K) {
        const floatx4u lo = *reinterpret_cast<const floatx4u*>(xrow + k);
        const floatx4u hi = *reinterpret_cast<const floatx4u*>(xrow + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + q * 8 + i < p.K ? xrow[k + i] : 0.0f;
      }
      bf16x8 xs[3];
      split<3>(v, xs);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j >= tiles) break;
        bf16x8 ws[Wt::kTerms];
        w[j].terms(ws);
#pragma unroll
        for (int i = 0; i < kProducts<Wt::kTerms>; ++i)
          t[j] = mfma16(ws[weight_term<Wt::kTerms>(i)], xs[value_term<Wt::kTerms>(i)], t[j]);
      }
    }
    sums[0][wave][lane] = t[0];
    sums[1][wave][lane] = t[1];
    __syncthreads();  // (this one also keeps an adapter's inner values from the next's until all have read them)
    if (wave < 2) {
      floatx4 sum = sums[wave][0][lane];
#pragma unroll
      for (int i = 1; i < W; ++i) sum += sums[wave][i][lane];
      *reinterpret_cast<floatx4*>(&inner[(lane & 15) * kInner + wave * 16 + q * 4]) =
          wave < tiles ? sum * scale : floatx4{};
    }
    __syncthreads();
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = inner[(lane & 15) * kInner + q * 8 + i];
    bf16x8 ts[3];
    split<3>(v, ts);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      bf16x8 ws[Wt::kTerms];
      wu[j].terms(ws);
#pragma unroll
      for (int i = 0; i < kProducts<Wt::kTerms>; ++i)
        acc[j] = mfma16(ws[weight_term<Wt::kTerms>(i)], ts[value_term<Wt::kTerms>(i)], acc[j]);
    }
    if (mine) {
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[j] += yv[j];
      store(acc);
    }
  });
  if (p.out != p.y && blockIdx.z == 0 && m < p.M && row_rank <= 0) {  // rows without an adapter
    load_y();
    store(yv);
  }
}

// Whether both products go in one launch: where a column block's own sums are little work, and not many of them.  16
// rows of 16 adapters, 1024 -> 1024, rank 16: 7.1 us against 9.4; 64 rows of 64: 8.5 against 9.3; but 64 rows of 64,
// 1024 -> 6144, rank 32: 32 against 15, and 2 rows, 4096 -> 1024, rank 64: 37 against 13.
bool few_rows(int M, int K, int N, int R) {
  return R <= 32 && K <= 2048 && (M <= 16 || (M <= 64 && N <= 2048));
}
constexpr int kFewTiles = 2, kFewWaves = 8;
constexpr int kDownWaves = 8, kUpWaves = 4;
constexpr int kUnits = 256;  // compute units

// Row and rank tiles a workgroup of the first kernel, the parts that it splits K into, the workgroups that share a row
// tile's adapters, and the second kernel's column tiles a wave.
//   - Two row tiles read an adapter's values half as often: 12294 x 1024, rank 16: 15.3 us against 16.9 (four: 15.6, and
//     20 where requests meet, since a workgroup that fills a compute unit by itself then ends last).  But half as many
//     workgroups go through twice as many adapters one after the other where requests meet: 4380 x 1181, rank 25, 222
//     requests: 36 us, 22 with one; 2100 x 4096, rank 128 in fp32, 4 adapters: 56, 36 with one.  So a bank of one slot
//     takes them sooner, and with large ranks sooner still (that call with one adapter: 45 us, one row tile 60; rank 64,
//     4000 x 4096: 40, one 39).
//   - With two row tiles the border between requests in a pass of its own.  It pays while a border's workgroup, which
//     takes twice its time, would end last, and adds a turn of workgroups that mostly end at once: where borders are
//     many (slots) or the rounds few.  K 1024, fp32, rank 64, without and with: 7100 rows of 2 requests 23.0, 21.5 us;
//     12294: 35.7, 33.2; 16384: 37.0, 39.7; 33000: 71.2, 74.8; of 12 requests in 4 slots 7100: 26.9, 24.7; 16500: 39.7,
//     38.1; 33000: 59.0, 61.2.  Where it just overfills a round it still gains for most requests (8192 rows: 4 % slower
//     of 2 requests, 4 to 14 % faster of 12 to 256).
//   - Eight rank tiles, which read x once, only there and not for fp32's three planes, whose 96 registers are too many
//     (16384 x 1024, rank 128: bf16 38 -> 26 us, fp16 52 -> 42; one row tile: fp16 45 -> 53).
//   - Few rows leave the chip idle without the next two: 64 rows of an adapter each, K 1024 -> N 6144, rank 32, take 68
//     + 17 us with one workgroup a tile, 6.8 + 8.1 with 16 and 8.  Parts of K past that cost the second kernel more
//     (1000 x 4096 x 4096, rank 128: two parts 44 us, four 57).
//   - Eight column tiles read t and each adapter's border least, from where the waves come in many rounds (8202 x 6144:
//     109 us, four 117; 12294 x 2900: 91, 98; but 14644 x 1743: 54, 49).  Two where few waves leave the chip idle (of 4
//     adapters, rank 16: 300 x 600 7.9 us, four 8.4; 130 x 3000 7.9, 8.5; 130 x 5000 8.1, 8.7; rank 32 in fp16: 3000 x
//     400 12.3, 11.7; 300 x 6000 12.0, 11.2).  A wave takes a turn for each adapter of its rows and loads their numbers
//     and inner values anew, so those count as waves too, as many as slots spread over the rows let expect (of 64
//     adapters, rank 32 in fp16: 64 x 6144 14.5 us, four 13.8; 64 x 3000 12.7, 11.9; 130 x 3000 11.9, 11.7; but 300 x
//     600 9.8, 9.9).  Many parts of K make each wave add up t again (336 rows, 3099 -> 1046, six parts: 18.2, four 13.3).
struct Plan {
  int row_tiles, rank_tiles, splits, down_passes, column_tiles, up_passes;
};

Plan plan_of(int M, int K, int N, int slots, int R, int dtype) {
  const int tiles = ceil_div(R, 16), most = std::min({16, M, slots}), row_tiles = ceil_div(M, 16);
  Plan pl{1, 4, 1, 1, 4, 1};
  if (slots > 1 ? M > 6144 : M > 4096 || (M > 2048 && R > 64)) pl.row_tiles = 2;
  if (tiles <= 2)
    pl.rank_tiles = tiles;
  else if (tiles > 4 && pl.row_tiles == 2 && dtype != kAdapterF32)
    pl.rank_tiles = 8;
  const int workgroups = ceil_div(M, 16 * pl.row_tiles) * ceil_div(tiles, pl.rank_tiles);
  pl.splits = std::max(1, std::min({kUnits / workgroups, ceil_div(K, 32) / (2 * kDownWaves), 8}));
  if (pl.row_tiles == 1)
    pl.down_passes = std::max(1, std::min(1024 / (workgroups * pl.splits), most));
  else if (slots > 1 && workgroups < kUnits * std::min(slots, 4))
    pl.down_passes = 2;
  const int64_t waves = (int64_t)row_tiles * ceil_div(N, 64);
  const int adapters = std::clamp((int)(INT64_C(16) * slots / M), 1, most);  // of a row tile
  if (waves * adapters < 3 * kUnits && pl.splits <= 2)
    pl.column_tiles = 2;
  else if (waves >= 32768)
    pl.column_tiles = 8;
  const int64_t shares = (int64_t)row_tiles * ceil_div(N, 16 * pl.column_tiles * kUpWaves);
  pl.up_passes = (int)std::max<int64_t>(1, std::min<int64_t>(1024 / shares, most));
  return pl;
}

template <int DTYPE, int RT>
void launch_down(const LowRankParams& p, const Plan& pl, hipStream_t stream) {
  auto run = [&](auto rb) {
    constexpr int RB = decltype(rb)::value;
    const int blocks = ceil_div(ceil_div(p.R, 16), RB);
    low_rank_down_kernel<DTYPE, RT, RB, kDownWaves>
        <<<dim3(ceil_div(p.M, 16 * RT), blocks * pl.splits, pl.down_passes), kDownWaves * 64, 0, stream>>>(
            p, blocks, pl.splits, pl.down_passes);
  };
  if constexpr (RT == 2 && DTYPE != kAdapterF32) {
    if (pl.rank_tiles == 8) return run(std::integral_constant<int, 8>{});
  }
  if (pl.rank_tiles == 1)
    run(std::integral_constant<int, 1>{});
  else if (pl.rank_tiles == 2)
    run(std::integral_constant<int, 2>{});
  else
    run(std::integral_constant<int, 4>{});
}

template <int DTYPE, int NT>
void launch_up(const LowRankParams& p, const Plan& pl, hipStream_t stream) {
  const int row_blocks = ceil_div(p.M, 16), rows = std::min(row_blocks, 65535);
  const dim3 grid(ceil_div(p.N, 16 * NT * kUpWaves), rows,
                  pl.up_passes > 1 ? pl.up_passes : ceil_div(row_blocks, rows));
  low_rank_up_kernel<DTYPE, NT, kUpWaves><<<grid, kUpWaves * 64, 0, stream>>>(p, pl.splits, pl.up_passes);
}

template <int DTYPE>
void launch_typed(const LowRankParams& p, hipStream_t stream) {
  if (few_rows(p.M, p.K, p.N, p.R)) {
    const int passes = std::min({16, p.M, p.slots});
    low_rank_few_kernel<DTYPE, kFewTiles, kFewWaves>
        <<<dim3(ceil_div(p.N, 16 * kFewTiles * kFewWaves), ceil_div(p.M, 16), passes), kFewWaves * 64, 0, stream>>>(
            p, passes);
    return;
  }
  const Plan pl = plan_of(p.M, p.K, p.N, p.slots, p.R, DTYPE);
  if (pl.row_tiles == 1)
    launch_down<DTYPE, 1>(p, pl, stream);
  else
    launch_down<DTYPE, 2>(p, pl, stream);
  if (pl.column_tiles == 2)
    launch_up<DTYPE, 2>(p, pl, stream);
  else if (pl.column_tiles == 4)
    launch_up<DTYPE, 4>(p, pl, stream);
  else
    launch_up<DTYPE, 8>(p, pl, stream);
}

}  // namespace

int64_t low_rank_scratch_bytes(int M, int K, int N, int slots, int R, int dtype) {
  if (few_rows(M, K, N, R)) return 0;
  return 4 * (meta_floats(M) + (int64_t)plan_of(M, K, N, slots, R, dtype).splits * M * ceil_div(R, 16) * 16);
}

int launch_low_rank_add(const LowRankParams& p, hipStream_t stream) {
  switch (p.dtype) {
    case kAdapterF32: launch_typed<kAdapterF32>(p, stream); break;
    case kAdapterBf16: launch_typed<kAdapterBf16>(p, stream); break;
    default: launch_typed<kAdapterF16>(p, stream); break;
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace tsplat
