// Device side of the 8-bit rows, shared by the kernels that make them and those that multiply them.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "fp8.h"
#include "tsplat_common.h"

namespace tsplat {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef _Float16 half_t;

template <class T>
struct Vec4;
template <>
struct Vec4<float> {
  typedef float type __attribute__((ext_vector_type(4)));
};
template <>
struct Vec4<bf16_t> {
  typedef bf16_t type __attribute__((ext_vector_type(4)));
};
template <>
struct Vec4<half_t> {
  typedef half_t type __attribute__((ext_vector_type(4)));
};

// Values 4 at a time from k on, zero past K; VEC: the row's quadruples are aligned to their size.
template <class T, bool VEC>
__device__ __forceinline__ floatx4 load4(const T* row, int k, int K) {
  floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (VEC && k + 4 <= K) {
    const typename Vec4<T>::type u = *reinterpret_cast<const typename Vec4<T>::type*>(row + k);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i < K) v[i] = (float)row[k + i];
  }
  return v;
}

// The bits of the largest finite magnitude of a lane's COUNT quadruples and of its neighbours' by `over`, which agrees on
// the largest of a float's bits.  Values that are not finite are rare: only a wave that meets an infinity looks at each
// value (a NaN is passed over by the maximum).
template <int COUNT, class Over>
__device__ __forceinline__ uint32_t largest_bits(const floatx4 (&v)[COUNT], Over over) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < COUNT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[i][e]));
  uint32_t bits = over(__float_as_uint(top));
  if (__any(bits >= 0x7f800000u)) {
    bits = 0;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = __float_as_uint(v[i][e]) & 0x7fffffffu;
        bits = max(bits, u < 0x7f800000u ? u : 0u);
      }
    bits = over(bits);
  }
  return bits;
}

// The exponent (+ 127) of the block's scale from its largest magnitude's bits: the smallest e with
// largest / 2^e <= 448 = 1.75 * 2^8, at least -127; 0 for a block of zeros.
__device__ __forceinline__ int scale_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top == 0 ? 127 : max(e, 0);
}

// 2^-(e - 127), a normal number: e is 247 at most.
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }

// Four codes of v * inverse.  The product is exact (a subnormal one is far below half of the smallest code), so there
// is one rounding, the conversion's, to nearest even; 448 is never passed by a finite value.  An infinity becomes a NaN
// like a NaN (the conversion makes 448 of it).
__device__ __forceinline__ int encode4(const floatx4& v, float inverse) {
  float u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = v[i] * inverse;
  if (__any(!(fmaxf(fmaxf(fabsf(u[0]), fabsf(u[1])), fmaxf(fabsf(u[2]), fabsf(u[3]))) <= 448.0f))) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = fabsf(u[i]) <= 448.0f ? u[i] : __uint_as_float(0x7fc00000u);
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], w, true);
}

}  // namespace tsplat
