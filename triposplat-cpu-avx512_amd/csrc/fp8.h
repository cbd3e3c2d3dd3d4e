// 8-bit rows: e4m3 codes with a power-of-two scale for each block of 128 of a row (include/tsplat_hip_fp8.h), and the
// host-side launches on them.  Every launcher assumes arguments that its caller has checked.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tsplat {

enum ValueType : int { kValueF32 = 0, kValueBf16 = 1, kValueF16 = 2 };

constexpr int kFp8Block = 128;
// Bytes of a row's codes, and of its exponents (a lane takes four of them as one dword).
inline int64_t fp8_code_stride(int64_t K) { return (K + kFp8Block - 1) / kFp8Block * kFp8Block; }
inline int64_t fp8_exponent_stride(int64_t K) { return (fp8_code_stride(K) / kFp8Block + 3) / 4 * 4; }

struct Fp8QuantizeParams {
  const void* x;
  int dtype;
  int64_t x_stride;
  int rows, K;
  uint8_t* codes;
  uint8_t* exponents;
};
int launch_fp8_quantize(const Fp8QuantizeParams& p, hipStream_t stream);

struct Fp8LinearParams {
  const void* x;  // or null: x_codes, x_exponents
  int x_dtype;
  int64_t x_stride;
  const uint8_t* x_codes;
  const uint8_t* x_exponents;
  const uint8_t* w_codes;
  const uint8_t* w_exponents;
  const float* bias;  // or null
  int activation;     // 1: gelu_tanh
  const float* gate;  // or null
  int64_t gate_stride, rows_per_batch;
  const void* residual;  // or null, of out_dtype
  int64_t residual_stride;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int M, K, N;
  uint8_t* scratch;
};
int64_t fp8_linear_scratch_bytes(int M, int K, int N, bool x_given);
int launch_fp8_linear(const Fp8LinearParams& p, hipStream_t stream);

}  // namespace tsplat
