// C-ABI of the 8-bit rows and products (include/tsplat_hip_fp8.h): argument checks and extents, then the launch on the
// caller's stream.  Nothing here allocates or waits.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "capi_spans.h"
#include "fp8.h"
#include "../../include/tsplat_hip_fp8.h"

using namespace tsplat;

namespace {

constexpr int kFp8AbiVersion = 1;
constexpr int kMaxRows = 1 << 27, kMaxFeatures = 1 << 20;  // (the launches' grids and 32-bit columns hold these)

int launched(int st) {
  if (st == kErrLaunch) (void)note(hipErrorLaunchFailure);
  return st;
}

bool within(int n, int most) { return n > 0 && n <= most; }
bool is_type(int t) { return t == kValueF32 || t == kValueBf16 || t == kValueF16; }
int size_of(int t) { return t == kValueF32 ? 4 : 2; }

}  // namespace

extern "C" {

int tsplat_fp8_abi_version(void) { return kFp8AbiVersion; }

int tsplat_fp8_quantize_async(const void* x, int dtype, int64_t x_stride, int rows, int K, uint8_t* codes,
                              uint8_t* exponents, void* stream) {
  if (!x || !codes || !exponents) return kErrNull;
  if (!within(rows, kMaxRows) || !within(K, kMaxFeatures) || !is_type(dtype)) return kErrDims;
  if (!sane_rows(x_stride, rows, K)) return kErrRange;
  const Span in = span_rows(x, x_stride, rows, K, size_of(dtype));
  const Span c = span_whole(codes, rows * fp8_code_stride(K)), e = span_whole(exponents, rows * fp8_exponent_stride(K));
  if (!apart(c, in) || !apart(e, in) || !apart(c, e)) return kErrRange;
  if (!aligned_to(x, size_of(dtype)) || !aligned16(codes) || !aligned_to(exponents, 4)) return kErrAlign;
  DeviceRanges ptrs;
  TSPLAT_CHECK(ptrs.check(x, in.bytes()));
  TSPLAT_CHECK(ptrs.check(codes, c.bytes()));
  TSPLAT_CHECK(ptrs.check(exponents, e.bytes()));
  return launched(launch_fp8_quantize({x, dtype, rows == 1 ? 0 : x_stride, rows, K, codes, exponents},
                                      static_cast<hipStream_t>(stream)));
}

int64_t tsplat_fp8_linear_scratch_bytes(int M, int K, int N, int x_given) {
  if (!within(M, kMaxRows) || !within(K, kMaxFeatures) || !within(N, kMaxFeatures)) return 0;
  return fp8_linear_scratch_bytes(M, K, N, x_given != 0);
}

int tsplat_fp8_linear_async(const void* x, int x_dtype, int64_t x_stride, const uint8_t* x_codes,
                            const uint8_t* x_exponents, const uint8_t* w_codes, const uint8_t* w_exponents,
                            const float* bias, int activation, const float* gate, int64_t gate_stride,
                            int64_t rows_per_batch, const void* residual, int64_t residual_stride, void* out,
                            int out_dtype, int64_t out_stride, int M, int K, int N, void* scratch,
                            int64_t scratch_bytes, void* stream) {
  if (!w_codes || !w_exponents || !out || (!x && (!x_codes || !x_exponents))) return kErrNull;
  if (!within(M, kMaxRows) || !within(K, kMaxFeatures) || !within(N, kMaxFeatures) || !is_type(out_dtype) ||
      (x && !is_type(x_dtype)) || (activation != 0 && activation != 1))
    return kErrDims;
  const int xs = x ? size_of(x_dtype) : 1, os = size_of(out_dtype);
  if ((x && !sane_rows(x_stride, M, K)) || !sane_rows(out_stride, M, N) ||
      (residual && !sane_rows(residual_stride, M, N)))
    return kErrRange;
  if (gate && rows_per_batch <= 0) return kErrRange;
  const int64_t per = gate ? std::min<int64_t>(rows_per_batch, M) : M;
  const int64_t gates = gate_stride == 0 ? 1 : (M + per - 1) / per;  // (a stride of 0: one row for every batch entry)
  if (gate && !sane_rows(gate_stride, gates, N)) return kErrRange;
  const Span so = span_rows(out, out_stride, M, N, os);
  const Span sx = x ? span_rows(x, x_stride, M, K, xs) : span_whole(x_codes, M * fp8_code_stride(K));
  const Span se = span_whole(x ? nullptr : x_exponents, M * fp8_exponent_stride(K));
  const Span sr = span_rows(residual, residual_stride, M, N, os);
  // all that is read, the residual apart
  const Span reads[] = {sx, se, span_whole(w_codes, N * fp8_code_stride(K)),
                        span_whole(w_exponents, N * fp8_exponent_stride(K)), span_whole(bias, (int64_t)N * 4),
                        span_rows(gate, gate_stride, gates, N, 4)};
  const int64_t need = fp8_linear_scratch_bytes(M, K, N, x != nullptr);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need)) return kErrWorkspace;
  const Span room = span_whole(need > 0 ? scratch : nullptr, need);
  for (const Span& r : reads)
    if (r.p && (!apart(so, r) || (room.p && !apart(room, r)))) return kErrRange;
  if (residual && !same_rows(so, sr) && !apart(so, sr)) return kErrRange;
  if (room.p && (!apart(room, so) || (residual && !apart(room, sr)))) return kErrRange;
  if ((x && !aligned_to(x, xs)) || !aligned_to(out, os) || !aligned_to(residual, os) || !aligned_to(bias, 4) ||
      !aligned_to(gate, 4) || !aligned16(w_codes) || !aligned_to(w_exponents, 4) || !aligned16(scratch) ||
      (!x && (!aligned16(x_codes) || !aligned_to(x_exponents, 4))))
    return kErrAlign;
  DeviceRanges ptrs;
  TSPLAT_CHECK(ptrs.check(out, so.bytes()));
  if (residual && residual != out) TSPLAT_CHECK(ptrs.check(residual, sr.bytes()));
  for (const Span& r : reads)
    if (r.p) TSPLAT_CHECK(ptrs.check(r.p, r.bytes()));
  if (room.p) TSPLAT_CHECK(ptrs.check(room.p, need));
  Fp8LinearParams p{x, x_dtype, x_stride, x_codes, x_exponents, w_codes, w_exponents, bias, activation,
                    gate, gate_stride, per, residual, residual_stride, out, out_dtype, out_stride,
                    M, K, N, static_cast<uint8_t*>(scratch)};
  if (M == 1) p.x_stride = p.residual_stride = p.out_stride = 0;
  return launched(launch_fp8_linear(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
