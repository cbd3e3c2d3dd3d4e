// Rows to 8 bits: a block of 128 values of a row becomes e4m3 codes and the exponent of one power-of-two scale,
//   e = the smallest with max |x| <= 448 * 2^e,  code = e4m3(x / 2^e).
// One pass: 32 lanes read a block (4 values each), agree on its largest magnitude in registers and write 4 codes each.
// Bound by HBM: b + 1 bytes a value.  16384 x 4096 in fp32: 58 us, 5.8 TB/s read and written (a 1 GiB device copy: 5.0);
// in bf16 and fp16 46 us, 4.4 TB/s (a lane's loads are 8 bytes there).
// Blocks of a workgroup are asked for four at a time; 3 x 1001 in fp16 takes 3.7 us, a launch (the call 11, the host).

#include <algorithm>

#include "fp8_device.h"

namespace tsplat {
namespace {

constexpr int kThreads = 256, kGroups = kThreads / 32;
constexpr int kAhead = 4;  // blocks that 32 lanes ask for before they use the first

// A workgroup takes rows_per whole rows.
template <class T, bool VEC>
__global__ __launch_bounds__(kThreads) void fp8_quantize_kernel(Fp8QuantizeParams p, int rows_per, int code_stride,
                                                                int exp_stride) {
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int64_t row0 = (int64_t)blockIdx.x * rows_per;
  const int rows = (int)min((int64_t)rows_per, p.rows - row0);
  const uint32_t items = (uint32_t)rows * (uint32_t)exp_stride;
  const int blocks = code_stride / kFp8Block;
  const T* x = static_cast<const T*>(p.x) + row0 * p.x_stride;
  uint8_t* codes = p.codes + row0 * code_stride;
  uint8_t* exps = p.exponents + row0 * exp_stride;
  for (uint32_t i0 = group; i0 < items; i0 += kGroups * kAhead) {
    floatx4 v[kAhead];
    uint32_t row[kAhead];
    int block[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t i = i0 + j * kGroups;
      row[j] = i / (uint32_t)exp_stride;
      block[j] = (int)(i - row[j] * (uint32_t)exp_stride);
      v[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      if (i < items && block[j] < blocks)
        v[j] = load4<T, VEC>(x + row[j] * p.x_stride, block[j] * kFp8Block + lane * 4, p.K);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kGroups >= items) break;
      const floatx4 one[1] = {v[j]};
      const uint32_t top = largest_bits(one, [](uint32_t bits) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, d, 32));
        return bits;
      });
      const int e = scale_exponent(top);
      if (block[j] < blocks)
        *reinterpret_cast<int*>(codes + (int64_t)row[j] * code_stride + block[j] * kFp8Block + lane * 4) =
            encode4(v[j], inverse_scale(e));
      if (lane == 0) exps[(int64_t)row[j] * exp_stride + block[j]] = (uint8_t)e;
    }
  }
}

template <class T>
int launch(const Fp8QuantizeParams& p, hipStream_t stream) {
  const int code_stride = (int)fp8_code_stride(p.K), exp_stride = (int)fp8_exponent_stride(p.K);
  // (a launch's threads are counted in 32 bits: more rows to a workgroup for very many)
  const int rows_per = std::max({1, kGroups * kAhead / exp_stride, (p.rows >> 23) + 1});
  const dim3 grid((p.rows + rows_per - 1) / rows_per);
  const bool vec = reinterpret_cast<uintptr_t>(p.x) % (4 * sizeof(T)) == 0 && (p.rows == 1 || p.x_stride % 4 == 0);
  if (vec)
    fp8_quantize_kernel<T, true><<<grid, kThreads, 0, stream>>>(p, rows_per, code_stride, exp_stride);
  else
    fp8_quantize_kernel<T, false><<<grid, kThreads, 0, stream>>>(p, rows_per, code_stride, exp_stride);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace

int launch_fp8_quantize(const Fp8QuantizeParams& p, hipStream_t stream) {
  switch (p.dtype) {
    case kValueF32: return launch<float>(p, stream);
    case kValueBf16: return launch<bf16_t>(p, stream);
    default: return launch<half_t>(p, stream);
  }
}

}  // namespace tsplat
