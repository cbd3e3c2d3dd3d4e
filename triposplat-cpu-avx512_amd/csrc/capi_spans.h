// Rows in memory and whether two sets of them overlap, in bytes: for the entries whose arrays are of several types.
#pragma once

#include <stdint.h>

#include "capi_internal.h"
#include "tsplat_common.h"

namespace tsplat {

struct Span {
  const void* p;
  int64_t stride, rows, row;  // bytes from row to row, rows, bytes of a row
  int64_t bytes() const { return (rows - 1) * stride + row; }
};

// `values` of `size` bytes in each of `rows` rows that lie `stride` values apart; rows >= 1.
inline Span span_rows(const void* p, int64_t stride, int64_t rows, int64_t values, int size) {
  return {p, rows == 1 ? values * size : stride * size, rows, values * size};
}
inline Span span_whole(const void* p, int64_t bytes) { return {p, bytes, 1, bytes}; }

// Rows that do not overlap, and a size far from the end of 64 bits; stride in values.
inline bool sane_rows(int64_t stride, int64_t rows, int64_t values) {
  return rows == 1 || (stride >= values && stride <= (INT64_C(1) << 56) / rows);
}

inline bool same_rows(const Span& a, const Span& b) { return a.p == b.p && (a.rows == 1 || a.stride == b.stride); }

// Whether no byte belongs to both: apart as a whole, or column ranges of the same wider rows.
inline bool apart(const Span& a, const Span& b) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + (uintptr_t)a.bytes() <= pb || pb + (uintptr_t)b.bytes() <= pa) return true;
  if (a.rows == 1 || b.rows == 1 || a.stride != b.stride) return false;
  int64_t at = (int64_t)(pb - pa) % a.stride;  // b's first byte within a's rows
  if (at < 0) at += a.stride;
  return at >= a.row && at + b.row <= a.stride;
}

inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace tsplat
