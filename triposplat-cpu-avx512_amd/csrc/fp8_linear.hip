// A Linear on 8-bit rows and weights:  out = f(x8 w8^T + bias) * gate + residual,  f the tanh form of GELU or nothing.
//
// Both operands are e4m3 codes with a power-of-two scale for each 128 of a row: products of codes are exact, the scales
// are taken by the instructions that widen or multiply the codes, and the sums stay in fp32 registers.  The operands'
// lane layout along K does not matter as long as both agree (a sum has no order of its own).
// The weights are the first operand: a lane then holds four neighbouring columns of one row of the result.
//
// What bounds it, and measured (with the rows' conversion, which is HBM's time: 17 and 58 us of these):
// 16384x1024x4096 in fp32 with GELU 181 us, 16384x4096x1024 onto a gated residual 188: products through bf16 at 1.18
// PFLOP/s, what the matrix cores hold at their clock under that load (a library's 8192^3 in bf16: 1.12), and the result's
// bytes, which the products hide in part (the former 149 us, 40 of them its 268 MB).  Without the conversions to bf16 6
// us less, without the copies into LDS 9.  8-bit products (results of 16 bits): 16384x4096x4096 323 us, 1.70 PFLOP/s
// (a library's: 2.64), and 52 the conversion; 4101x1024x2048 28 us, of which 6 convert the rows and 10 are a launch and its
// chain of loads.  One row of 1024x1024 4.4 us (the call 11: the host), 64 rows of 1024x6144 13.  77 to 1370 rows of
// 1024x1024 18 us, of 4096x1024 42 to 48: 8 to 88 workgroups, each the whole of K long.

#include <algorithm>

#include "fp8_device.h"
#include "tsplat_launch.h"

namespace tsplat {
namespace {

// What follows the sums.
struct Finish {
  const float* bias;
  const float* gate;
  const void* residual;
  void* out;
  int64_t gate_stride, rows_per_batch, residual_stride, out_stride;
  int M, N, activation;
};

// y / (1 + exp(-2 u)), u = sqrt(2/pi) (y + 0.044715 y^3): 0.5 y (1 + tanh u) without its cancellation.  One hardware
// exp2 and reciprocal, 1 ulp each (the reference-named GELU kernels' polynomial and division take six times as long,
// more than the product at K = 1024).
__device__ __forceinline__ float gelu(float y) {
  constexpr float kA = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  const float u = y * fmaf(0.044715f * y, y, 1.0f);
  return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(kA * u));
}

// Columns n .. n + 3 of a row of N.  VEC: N is a multiple of 4 and columns in fours are aligned in everything that is
// read and written here (past N then: the last four, so that no lane's loads hang on a test); else zero past N.
template <class T, bool VEC>
__device__ __forceinline__ floatx4 columns4(const T* row, int n, int N) {
  return VEC ? load4<T, true>(row, min(n, N - 4), N) : load4<T, false>(row, n, N);
}

// The gate's row of row m.
__device__ __forceinline__ const float* gate_row(const Finish& f, int m) {
  return f.gate + (f.gate_stride ? (uint32_t)m / (uint32_t)f.rows_per_batch * f.gate_stride : 0);
}

// What follows the sums of columns n .. n + 3 in COUNT rows m(i); none is written past row M or column N.  bias: of these
// columns.  All of a piece's rows are asked for before the first is used.
template <class TO, bool VEC, int COUNT, class Rows>
__device__ __forceinline__ void finish(const Finish& f, floatx4 (&y)[COUNT], const floatx4& bias, int n, Rows m) {
  floatx4 gate[COUNT], residual[COUNT];
  if (f.gate) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) gate[i] = columns4<float, VEC>(gate_row(f, min(m(i), f.M - 1)), n, f.N);
  }
  if (f.residual) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      residual[i] = columns4<TO, VEC>(
          static_cast<const TO*>(f.residual) + (int64_t)min(m(i), f.M - 1) * f.residual_stride, n, f.N);
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i) y[i] += bias;
  if (f.activation) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][e] = gelu(y[i][e]);
  }
  if (f.gate) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) y[i] *= gate[i];
  }
  if (f.residual) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) y[i] += residual[i];
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if (m(i) >= f.M) continue;
    TO* out = static_cast<TO*>(f.out) + (int64_t)m(i) * f.out_stride;
    if constexpr (VEC) {
      typename Vec4<TO>::type o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (TO)y[i][e];
      if (n < f.N) *reinterpret_cast<typename Vec4<TO>::type*>(out + n) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < f.N) out[n + e] = (TO)y[i][e];
    }
  }
}

template <bool VEC>
__device__ __forceinline__ floatx4 bias_of(const Finish& f, int n) {
  return f.bias ? columns4<float, VEC>(f.bias, n, f.N) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
}

__device__ __forceinline__ intx8 join(const intx4& a, const intx4& b) {
  return intx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A wave's copy from memory to LDS, lane i's 16 (4) bytes to `to` + 16 i (4 i); `to` is the same for all lanes.  Written
// as instructions because the compiler, which cannot tell the buffers apart, else waits for every copy under way before
// each read of LDS.  wait_and_meet orders them.  (M0, which holds the place, has no other use here.)
__device__ __forceinline__ uint32_t lds_place(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
__device__ __forceinline__ void copy16_to_lds(const uint8_t* from, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds_place(to)) : "memory");
}
__device__ __forceinline__ void copy4_to_lds(const uint8_t* from, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds_place(to)) : "memory");
}

// Waits until at most N of this wave's memory operations are under way and its reads of LDS are done, then for the
// workgroup's other waves: what they all copied before the last N operations is in LDS, and what they read may be
// overwritten.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  static_assert(N < 64, "the counter's range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Workgroup i runs on XCD i % 8: the tiles of one XCD become neighbours.
__device__ __forceinline__ int tile_of(int id, int count) {
  const int per = count / 8, more = count % 8, xcd = id % 8;
  return xcd * per + min(xcd, more) + id / 8;
}

// One step of the products over a lane's 32 codes of a row (two pieces of 16) with the scale's exponent, for rows of
// weights (w) and of x.  EXACT: the codes, scaled, as bf16 (exact) through v_mfma_f32_32x32x16_bf16, whose sums are fp32.
// Otherwise as they are through v_mfma_scale_f32_32x32x64_f8f6f4, at twice that rate, which brings each 8 neighbouring
// products to the largest one's exponent and cuts them there at 2^-13 of its power of two: a relative error of about
// 1.5e-5 of a sum, far below the rounding of a 16-bit result and too much for an fp32 one.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 2^(e - 127): the conversions below take the scale's exponent field alone, 0 among its values.
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float((e & 0xffu) << 23); }

// Eight codes as bf16, times the scale: exact down to 2^-126, below that to bf16's smallest step of 2^-133.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- many rows: tiles of BM x BN through LDS, STAGES buffers of 64 codes of each row.
// A row's 64 bytes are pieces of 16, and a wave reads one piece of each of 32 rows at once, eight lanes (rows) in a cycle
// of all banks: piece c of row r lies at place c ^ (r / 2 % 4).  The copies to LDS write in lane order, so the lane picks
// its piece.
// A stage is multiplied in two steps, of 32 codes each (EXACT) or of half of the weights' rows.  The operands of each step
// are read into registers while the one before is multiplied, so a stage's buffer is free, and the copies of the stage that
// comes STAGES later may begin, before its last step is multiplied.
// 128x256 tiles, two workgroups a CU; 128x128 where there are fewer than two of the wide ones for each CU (4101x1024x2048:
// 23 against 25 us; 16384x1024x4096 in 16 bits the wide ones, half the reads of x).
constexpr int kStage = 64;

template <int BM, int BN, int WM, int WN, int STAGES, class TO, bool VEC>
__global__ __launch_bounds__(WM* WN * 64, BM * BN > 128 * 128 ? 2 : 3) void fp8_tile_kernel(const uint8_t* __restrict__ xc,
                                                                  const uint8_t* __restrict__ xe,
                                                                  const uint8_t* __restrict__ wc,
                                                                  const uint8_t* __restrict__ we, Finish f,
                                                                  int code_stride, int exp_stride, int tiles_n) {
  constexpr bool kExact = sizeof(TO) == 4;
  constexpr int kWaves = WM * WN, kPieces = kStage / 16, kRowsACopy = 64 / kPieces;
  constexpr int kCopies = (BM + BN) / kRowsACopy / kWaves;
  constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int NS = kExact ? NI : NI / 2;  // of the weights' 32 rows, in a step
  constexpr int kExpCopies = (BM + BN) / 64;
  static_assert((BM + BN) % 64 == 0 && BM % 64 == 0, "whole copies of exponents");
  static_assert(kCopies * kRowsACopy * kWaves == BM + BN && BM % kRowsACopy == 0, "whole copies");
  __shared__ __attribute__((aligned(16))) uint8_t lds[STAGES][(BM + BN) * kStage];
  __shared__ __attribute__((aligned(16))) uint8_t exps[2][(BM + BN) * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Wide tiles: bands of 16 row tiles, in them runs of 4 column tiles, whose operands stay in the XCD's L2 (16384x1024x4096
  // in fp32 163 -> 157 us, 16384x4096x4096 in bf16 5 % less); small ones, few enough, row after row.
  constexpr int kBand = BM * BN > 128 * 128 ? 16 : 1, kRun = 4;
  int tile = tile_of(blockIdx.x, gridDim.x), m0 = tile / tiles_n * BM, n0 = tile % tiles_n * BN;
  if constexpr (kBand > 1) {
    const int band = tile / (kBand * tiles_n), rows = min(kBand, (int)gridDim.x / tiles_n - band * kBand);
    tile -= band * kBand * tiles_n;
    const int run = tile / (rows * kRun), columns = min(kRun, tiles_n - run * kRun);
    tile -= run * rows * kRun;
    m0 = (band * kBand + tile / columns) * BM;
    n0 = (run * kRun + tile % columns) * BN;
  }
  const int blocks = code_stride / kFp8Block, stages = blocks * (kFp8Block / kStage);
  auto place = [](int r, int c) { return c ^ ((r >> 1) & 3); };

  const uint8_t* from[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int r = (j * kWaves + wave) * kRowsACopy + lane / kPieces;
    const int64_t row = r < BM ? min(m0 + r, f.M - 1) : min(n0 + r - BM, f.N - 1);  // (past the end: the last row)
    from[j] = (r < BM ? xc : wc) + row * code_stride + place(r, lane % kPieces) * 16;
  }
  // Exponents of four blocks of 128, a dword of each row.
  auto fetch_exps = [&](int four) {
#pragma unroll
    for (int j = 0; j < (kExpCopies + kWaves - 1) / kWaves; ++j) {
      const int r0 = (j * kWaves + wave) * 64;
      if (r0 >= BM + BN) break;
      const int r = r0 + lane;
      const int64_t row = r < BM ? min(m0 + r, f.M - 1) : min(n0 + r - BM, f.N - 1);
      copy4_to_lds((r < BM ? xe : we) + row * exp_stride + four * 4, &exps[four & 1][r0 * 4]);
    }
  };
  auto fetch = [&](int stage, int buffer) {
    if (stage % 8 == 0) fetch_exps(stage / 8);
#pragma unroll
    for (int j = 0; j < kCopies; ++j)
      copy16_to_lds(from[j] + stage * kStage, &lds[buffer][(j * kWaves + wave) * kRowsACopy * kStage]);
  };

  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int l32 = lane & 31, half = lane >> 5;
  const bool busy = m0 + wm < f.M && n0 + wn < f.N;  // (a ragged last tile: its waves without rows only copy)
  floatx16 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // A step's operands: pieces of the weights' rows and of x's, and the exponents of their block.
  struct Step {
    typedef std::conditional_t<kExact, intx4, intx8> Codes;
    Codes w[NS], x[MI];
  };
  struct Scales {
    uint32_t w[NI], x[MI];
  };
  auto read_step = [&](Step& to, int buffer, int step) {
    const uint8_t* a = &lds[buffer][(BM + wn + l32) * kStage];
    const uint8_t* b = &lds[buffer][(wm + l32) * kStage];
    auto codes = [&](const uint8_t* row) {
      const intx4 lo = *reinterpret_cast<const intx4*>(row + place(l32, (kExact ? 2 * step : 0) + half) * 16);
      if constexpr (kExact)
        return lo;
      else
        return join(lo, *reinterpret_cast<const intx4*>(row + place(l32, 2 + half) * 16));
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) to.w[i] = codes(a + ((kExact ? 0 : step * NS) + i) * 32 * kStage);
#pragma unroll
    for (int i = 0; i < MI; ++i) to.x[i] = codes(b + i * 32 * kStage);
  };
  auto read_scales = [&](Scales& to, int block) {
    const uint8_t* e = &exps[block >> 2 & 1][block & 3];
#pragma unroll
    for (int i = 0; i < NI; ++i) to.w[i] = e[(BM + wn + i * 32 + l32) * 4];
#pragma unroll
    for (int i = 0; i < MI; ++i) to.x[i] = e[(wm + i * 32 + l32) * 4];
  };
  auto multiply = [&](const Step& s, const Scales& q, int step) {
    if constexpr (kExact) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 wb[NI], xb[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) xb[i] = widen8(s.x[i][2 * h], s.x[i][2 * h + 1], scale_of(q.x[i]));
#pragma unroll
        for (int i = 0; i < NI; ++i) wb[i] = widen8(s.w[i][2 * h], s.w[i][2 * h + 1], scale_of(q.w[i]));
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < MI; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i], xb[j], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) {
          floatx16& c = acc[step * NS + i][j];
          c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(s.w[i], s.x[j], c, 0, 0, 0, (int)q.w[step * NS + i], 0,
                                                             (int)q.x[j]);
        }
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (i < stages) fetch(i, i);
  if (stages >= STAGES)
    wait_and_meet<(STAGES - 1) * kCopies>();
  else
    wait_and_meet<0>();
  Step now, next;
  Scales scales, scales_next;
  if (busy) read_step(now, 0, 0);
  read_scales(scales, 0);
  int buffer = 0;
  for (int block = 0; block < blocks; ++block) {
#pragma unroll
    for (int half_block = 0; half_block < 2; ++half_block) {
      const int stage = 2 * block + half_block;
      if (busy) {
        read_step(next, buffer, 1);
        multiply(now, scales, 0);
      }
      const int after = buffer == STAGES - 1 ? 0 : buffer + 1;
      if (stage + 1 < stages) {
        // The next stage's copies are done when at most those of the STAGES - 2 after it are under way (exponents are asked
        // for before the codes of their stage); this stage is in every wave's registers then.
        if (stage + STAGES - 1 < stages)
          wait_and_meet<(STAGES - 2) * kCopies>();
        else
          wait_and_meet<0>();
        if (busy) read_step(now, after, 0);
        if (half_block == 1) read_scales(scales_next, block + 1);
        if (stage + STAGES < stages) fetch(stage + STAGES, buffer);
      }
      if (busy) multiply(next, scales, 1);
      buffer = after;
    }
    scales = scales_next;
  }

  // A lane holds four columns of one row, 32 rows to a store: through LDS (a wave's 32 rows at a time, its own) a store
  // and the loads beside it take whole rows of the wave's tile instead.
  constexpr int kPitch = NI * 32 + 4, kLanesARow = NI * 8, kRowsAtOnce = 64 / kLanesARow,
                kBatch = NI * MI > 4 ? 8 : 4;  // (rows to a lane at once, as registers allow)
  static_assert(kWaves * 32 * kPitch * 4 <= (int)sizeof(lds), "the waves' rows fit");
  float* rows = reinterpret_cast<float*>(&lds[0][0]) + wave * 32 * kPitch;
  const int n = n0 + wn + lane % kLanesARow * 4, r0 = lane / kLanesARow;
  const floatx4 bias = bias_of<VEC>(f, n);
  __syncthreads();
  if (!busy) return;
#pragma unroll
  for (int j = 0; j < MI; ++j) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<floatx4*>(rows + l32 * kPitch + i * 32 + g * 8 + half * 4) =
            floatx4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
    __builtin_amdgcn_wave_barrier();
    for (int r = r0; r < 32; r += kBatch * kRowsAtOnce) {
      floatx4 y[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        y[i] = *reinterpret_cast<const floatx4*>(rows + (r + i * kRowsAtOnce) * kPitch + lane % kLanesARow * 4);
      finish<TO, VEC>(f, y, bias, n, [&](int i) { return m0 + wm + j * 32 + r + i * kRowsAtOnce; });
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- few rows (up to 64): bound by reading the weights once.  A workgroup takes 16 NB columns and all rows, its eight
// waves every eighth block of K each, straight from memory to registers; their sums meet in LDS.  x is brought to 8
// bits on the way (a lane holds 32 values of a row, four lanes its block of 128): one launch, no scratch.  Two column
// tiles from 17 rows on, which halves the workgroups that convert x (64 rows of 1024x6144 23 -> 13 us); one for a few
// rows, whose time is a chain of loads (4.4 us).  Products through bf16: their rate does not matter here.
constexpr int kFewWaves = 8;

template <class T, bool VEC, int MB, int NB, class TO, bool VECO>
__global__ __launch_bounds__(kFewWaves * 64) void fp8_few_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                 const uint8_t* __restrict__ xc,
                                                                 const uint8_t* __restrict__ xe,
                                                                 const uint8_t* __restrict__ wc,
                                                                 const uint8_t* __restrict__ we, Finish f, int K,
                                                                 int code_stride, int exp_stride) {
  __shared__ floatx4 part[kFewWaves][MB * NB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, quarter = lane >> 4;
  const int n0 = blockIdx.x * 16 * NB;
  const int blocks = code_stride / kFp8Block;
  const uint8_t* wrow[NB];
  const uint8_t* wexp[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int64_t n = min(n0 + i * 16 + l16, f.N - 1);
    wrow[i] = wc + n * code_stride + quarter * 32;
    wexp[i] = we + n * exp_stride;
  }
  floatx4 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int block = wave; block < blocks; block += kFewWaves) {
    intx8 wv[NB];
    int wq[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const intx4* at = reinterpret_cast<const intx4*>(wrow[i] + block * kFp8Block);
      wv[i] = join(at[0], at[1]);
      wq[i] = wexp[i][block];
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int64_t m = min(j * 16 + l16, f.M - 1);
      intx8 xv;
      int xq;
      if (x) {
        floatx4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = load4<T, VEC>(x + m * x_stride, block * kFp8Block + quarter * 32 + i * 4, K);
        const uint32_t top = largest_bits(v, [](uint32_t bits) {
          bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16));
          return max(bits, (uint32_t)__shfl_xor((int)bits, 32));
        });
        xq = scale_exponent(top);
#pragma unroll
        for (int i = 0; i < 8; ++i) xv[i] = encode4(v[i], inverse_scale(xq));
      } else {
        const intx4* at = reinterpret_cast<const intx4*>(xc + m * code_stride + block * kFp8Block + quarter * 32);
        xv = join(at[0], at[1]);
        xq = xe[m * exp_stride + block];
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const bf16x8 xb = widen8(xv[2 * h], xv[2 * h + 1], scale_of(xq));
#pragma unroll
        for (int i = 0; i < NB; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(wv[i][2 * h], wv[i][2 * h + 1], scale_of(wq[i])), xb,
                                                             acc[i][j], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) part[wave][i * MB + j][lane] = acc[i][j];
  __syncthreads();
  for (int t = threadIdx.x; t < MB * NB * 64; t += kFewWaves * 64) {
    const int at = t & 63, tile = t >> 6;
    const int m = tile % MB * 16 + (at & 15), n = n0 + tile / MB * 16 + (at >> 4) * 4;
    if (m >= f.M || n >= f.N) continue;
    floatx4 y[1] = {part[0][tile][at]};
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) y[0] += part[w][tile][at];
    finish<TO, VECO>(f, y, bias_of<VECO>(f, n), n, [&](int) { return m; });
  }
}

constexpr int kFewRows = 64;

bool in_fours(const void* p, int64_t stride, int64_t rows, int size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && (rows == 1 || stride % 4 == 0));
}

int size_of(int dtype) { return dtype == kValueF32 ? 4 : 2; }

template <class T, bool VEC, int MB, class TO>
int launch_few_rows(const Fp8LinearParams& p, const Finish& f, bool veco, hipStream_t stream) {
  constexpr int NB = MB >= 2 ? 2 : 1;
  const int grid = (p.N + 16 * NB - 1) / (16 * NB);
  auto go = [&](auto kernel) {
    kernel<<<grid, kFewWaves * 64, 0, stream>>>(static_cast<const T*>(p.x), p.x_stride, p.x_codes, p.x_exponents,
                                                p.w_codes, p.w_exponents, f, p.K, (int)fp8_code_stride(p.K),
                                                (int)fp8_exponent_stride(p.K));
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
  };
  return veco ? go(fp8_few_kernel<T, VEC, MB, NB, TO, true>) : go(fp8_few_kernel<T, VEC, MB, NB, TO, false>);
}

template <class T, class TO>
int launch_few(const Fp8LinearParams& p, const Finish& f, bool veco, hipStream_t stream) {
  const int mb = (p.M + 15) / 16;
  if (in_fours(p.x, p.x_stride, p.M, sizeof(T))) {
    if (mb == 1) return launch_few_rows<T, true, 1, TO>(p, f, veco, stream);
    if (mb == 2) return launch_few_rows<T, true, 2, TO>(p, f, veco, stream);
    return launch_few_rows<T, true, 4, TO>(p, f, veco, stream);
  }
  if (mb == 1) return launch_few_rows<T, false, 1, TO>(p, f, veco, stream);
  if (mb == 2) return launch_few_rows<T, false, 2, TO>(p, f, veco, stream);
  return launch_few_rows<T, false, 4, TO>(p, f, veco, stream);
}

template <int BM, int BN, int WM, int WN, int STAGES, class TO>
int launch_tiles(const Fp8LinearParams& p, const uint8_t* xc, const uint8_t* xe, const Finish& f, bool veco,
                 hipStream_t stream) {
  const int tiles_n = (p.N + BN - 1) / BN;
  const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * tiles_n;
  if (tiles * WM * WN * 64 > UINT32_MAX) return kErrDims;  // (a launch's threads in 32 bits)
  auto go = [&](auto kernel) {
    kernel<<<(int)tiles, WM * WN * 64, 0, stream>>>(xc, xe, p.w_codes, p.w_exponents, f, (int)fp8_code_stride(p.K),
                                                    (int)fp8_exponent_stride(p.K), tiles_n);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
  };
  return veco ? go(fp8_tile_kernel<BM, BN, WM, WN, STAGES, TO, true>)
              : go(fp8_tile_kernel<BM, BN, WM, WN, STAGES, TO, false>);
}

template <class TO>
int launch_out(const Fp8LinearParams& p, hipStream_t stream) {
  const Finish f{p.bias, p.gate, p.residual, p.out, p.gate_stride, p.rows_per_batch, p.residual_stride, p.out_stride,
                 p.M, p.N, p.activation};
  const int size = size_of(p.out_dtype);
  const bool veco = p.N % 4 == 0 && in_fours(p.bias, 0, 1, 4) && in_fours(p.gate, p.gate_stride, p.M, 4) &&
                    in_fours(p.residual, p.residual_stride, p.M, size) && in_fours(p.out, p.out_stride, p.M, size);
  if (p.M <= kFewRows) {
    if (p.x && p.x_dtype == kValueBf16) return launch_few<bf16_t, TO>(p, f, veco, stream);
    if (p.x && p.x_dtype == kValueF16) return launch_few<half_t, TO>(p, f, veco, stream);
    return launch_few<float, TO>(p, f, veco, stream);
  }
  const uint8_t *xc = p.x_codes, *xe = p.x_exponents;
  if (p.x) {
    uint8_t* codes = p.scratch;
    uint8_t* exps = p.scratch + p.M * fp8_code_stride(p.K);
    const int st = launch_fp8_quantize({p.x, p.x_dtype, p.x_stride, p.M, p.K, codes, exps}, stream);
    if (st != kOk) return st;
    xc = codes, xe = exps;
  }
  const int64_t wide = (int64_t)((p.M + 127) / 128) * ((p.N + 255) / 256);
  if (wide < 2 * compute_units()) return launch_tiles<128, 128, 2, 2, 3, TO>(p, xc, xe, f, veco, stream);
  return launch_tiles<128, 256, 2, 2, 3, TO>(p, xc, xe, f, veco, stream);
}

}  // namespace

int64_t fp8_linear_scratch_bytes(int M, int K, int N, bool x_given) {
  if (!x_given || M <= kFewRows) return 0;
  return (M * (fp8_code_stride(K) + fp8_exponent_stride(K)) + 15) / 16 * 16;
}

int launch_fp8_linear(const Fp8LinearParams& p, hipStream_t stream) {
  switch (p.out_dtype) {
    case kValueF32: return launch_out<float>(p, stream);
    case kValueBf16: return launch_out<bf16_t>(p, stream);
    default: return launch_out<half_t>(p, stream);
  }
}

}  // namespace tsplat
