// C-ABI of the operators that serve a batch of several requests (include/tsplat_hip_requests.h): argument checks
// and extents, then the launch on the caller's stream.  Nothing here allocates or waits.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "capi_internal.h"
#include "tsplat_common.h"
#include "tsplat_launch.h"
#include "../../include/tsplat_hip_requests.h"

using namespace tsplat;

namespace {

constexpr int kRequestsAbiVersion = 1;
constexpr int kMaxRank = 512;
constexpr int kMaxRows = 1 << 27, kMaxFeatures = 1 << 20;  // (the launches' grids hold these)
constexpr int kMaxSlots = 1 << 20;
constexpr int kMaxHeadDim = 512;
constexpr int kMaxHeads = 1 << 16;
constexpr int kMaxAxes = 8;

int launched(int st) {
  if (st == kErrLaunch) (void)note(hipErrorLaunchFailure);
  return st;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// A matrix of fp32 rows; sizes and strides positive, below 2^62 bytes in all.
struct Rows {
  const float* p;
  int64_t stride, rows, cols;
  int64_t bytes() const { return ((rows - 1) * stride + cols) * 4; }
};

// rows * stride floats stay far from the end of 64 bits.
bool sane(const Rows& r) {
  return r.rows == 1 || (r.stride >= r.cols && r.stride <= (INT64_C(1) << 60) / r.rows);
}

// Values in a row, `floats` of 4 bytes.
Rows whole(const void* p, int64_t floats) { return {static_cast<const float*>(p), floats, 1, floats}; }

bool same(const Rows& a, const Rows& b) { return a.p == b.p && (a.rows == 1 || a.stride == b.stride); }

// Whether no element belongs to both: apart as a whole, or column ranges of the same wider rows.
bool disjoint(const Rows& a, const Rows& b) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + (uintptr_t)a.bytes() <= pb || pb + (uintptr_t)b.bytes() <= pa) return true;
  if (a.rows == 1 || b.rows == 1 || a.stride != b.stride) return false;
  const int64_t bytes = a.stride * 4;
  int64_t at = (int64_t)(pb - pa) % bytes;  // b's first column within a's rows
  if (at < 0) at += bytes;
  return at >= a.cols * 4 && at + b.cols * 4 <= bytes;
}

bool low_rank_sizes(int M, int K, int N, int slots, int rank, int dtype) {
  auto within = [](int n, int most) { return n > 0 && n <= most; };
  return within(M, kMaxRows) && within(K, kMaxFeatures) && within(N, kMaxFeatures) && within(slots, kMaxSlots) &&
         within(rank, kMaxRank) && (dtype == kAdapterF32 || dtype == kAdapterBf16 || dtype == kAdapterF16);
}

}  // namespace

extern "C" {

int tsplat_requests_abi_version(void) { return kRequestsAbiVersion; }

int64_t tsplat_low_rank_scratch_bytes(int M, int K, int N, int slots, int max_rank, int dtype) {
  if (!low_rank_sizes(M, K, N, slots, max_rank, dtype)) return 0;
  return low_rank_scratch_bytes(M, K, N, slots, max_rank, dtype);
}

int tsplat_low_rank_add_async(const float* y, int64_t y_stride, const float* x, int64_t x_stride,
                              const int32_t* rows, const void* down, const void* up, const float* scale,
                              const int32_t* rank, float* out, int64_t out_stride, int M, int K, int N,
                              int slots, int max_rank, int dtype, void* scratch, int64_t scratch_bytes,
                              void* stream) {
  if (!y || !x || !rows || !down || !up || !scale || !rank || !out) return kErrNull;
  if (!low_rank_sizes(M, K, N, slots, max_rank, dtype)) return kErrDims;
  const Rows ry{y, y_stride, M, N}, rx{x, x_stride, M, K}, ro{out, out_stride, M, N};
  if (!sane(ry) || !sane(rx) || !sane(ro)) return kErrRange;
  if ((!same(ro, ry) && !disjoint(ro, ry)) || !disjoint(ro, rx)) return kErrRange;
  if (!aligned4(y) || !aligned4(x) || !aligned4(out) || !aligned4(rows) || !aligned4(scale) || !aligned4(rank) ||
      !aligned16(down) || !aligned16(up) || !aligned16(scratch))
    return kErrAlign;
  const int64_t need = low_rank_scratch_bytes(M, K, N, slots, max_rank, dtype);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need)) return kErrWorkspace;
  const int64_t size = dtype == kAdapterF32 ? 6 : 2;  // (fp32: three bf16 planes)
  const int64_t k_pad = ((int64_t)K + 31) / 32 * 32, n_pad = ((int64_t)N + 15) / 16 * 16;
  const int64_t down_values = ((int64_t)max_rank + 15) / 16 * 16 * k_pad;
  const int64_t up_values = ((int64_t)max_rank + 31) / 32 * 32 * n_pad;
  const Rows room = whole(need > 0 ? scratch : nullptr, need / 4);
  // what is only read besides y and x; y may be the output, but never scratch
  const Rows reads[] = {whole(rows, M), whole(down, slots * down_values * size / 4),
                        whole(up, slots * up_values * size / 4), whole(scale, slots), whole(rank, slots)};
  for (const Rows& r : reads)
    if (!disjoint(ro, r) || (room.p && !disjoint(room, r))) return kErrRange;
  if (room.p && (!disjoint(room, ry) || !disjoint(room, rx) || !disjoint(room, ro))) return kErrRange;
  DeviceRanges ptrs;
  TSPLAT_CHECK(ptrs.check(x, rx.bytes()));
  TSPLAT_CHECK(ptrs.check(y, ry.bytes()));
  TSPLAT_CHECK(ptrs.check(out, ro.bytes()));
  for (const Rows& r : reads) TSPLAT_CHECK(ptrs.check(r.p, r.bytes()));
  if (room.p) TSPLAT_CHECK(ptrs.check(scratch, need));
  LowRankParams p{y, x, rows, down, up, scale, rank, out, y_stride, x_stride, out_stride,
                  M, K, N, slots, max_rank, dtype, static_cast<float*>(scratch)};
  if (M == 1) p.y_stride = p.x_stride = p.out_stride = 0;
  return launched(launch_low_rank_add(p, static_cast<hipStream_t>(stream)));
}

int tsplat_residual_norm_async(const float* x, int64_t x_stride, const float* h, int64_t h_stride, float* out,
                               int64_t out_stride, float* normed, int64_t normed_stride, int64_t rows, int cols,
                               float residual_scale, const float* gate, int64_t gate_stride, int post_kind,
                               const float* post_weight, const float* post_bias, float post_eps, int pre_kind,
                               const float* pre_weight, const float* pre_bias, float pre_eps, const float* scale,
                               const float* shift, int64_t mod_stride, int64_t rows_per_batch, void* stream) {
  if (!x || !h || !out || !normed) return kErrNull;
  if (rows <= 0 || rows > INT32_MAX || cols <= 0 || !(post_eps >= 0.0f) || !(pre_eps >= 0.0f)) return kErrDims;
  if (post_kind != kNormNone && post_kind != kNormLayer && post_kind != kNormRms) return kErrDims;
  if (pre_kind != kNormLayer && pre_kind != kNormRms) return kErrDims;
  const Rows rx{x, x_stride, rows, cols}, rh{h, h_stride, rows, cols}, ro{out, out_stride, rows, cols},
      rn{normed, normed_stride, rows, cols};
  if (!sane(rx) || !sane(rh) || !sane(ro) || !sane(rn)) return kErrRange;
  const bool modulate = scale != nullptr || shift != nullptr;
  if (modulate && (!scale || !shift)) return kErrRange;
  if (post_kind == kNormNone && (post_weight || post_bias)) return kErrRange;
  if ((gate || modulate) && rows_per_batch <= 0) return kErrRange;
  const int64_t per = gate || modulate ? std::min(rows_per_batch, rows) : rows;
  const int64_t batches = (rows + per - 1) / per;
  // (a stride of 0: one row for every batch entry)
  const int64_t gates = gate_stride == 0 ? 1 : batches, mods = mod_stride == 0 ? 1 : batches;
  const Rows rg{gate, gate_stride, gates, cols}, rs{scale, mod_stride, mods, cols}, rt{shift, mod_stride, mods, cols};
  if ((gate && !sane(rg)) || (modulate && (!sane(rs) || !sane(rt)))) return kErrRange;
  if (!disjoint(ro, rn) || (!same(ro, rx) && !disjoint(ro, rx)) || !disjoint(ro, rh) || !disjoint(rn, rx) ||
      (!same(rn, rh) && !disjoint(rn, rh)))
    return kErrRange;
  // what is only read: the modulation's rows and the norms' vectors
  const Rows reads[] = {rg, rs, rt, Rows{post_weight, cols, 1, cols}, Rows{post_bias, cols, 1, cols},
                        Rows{pre_weight, cols, 1, cols}, Rows{pre_bias, cols, 1, cols}};
  for (const Rows& r : reads) {
    if (!r.p) continue;
    if (!disjoint(ro, r) || !disjoint(rn, r)) return kErrRange;
    if (!aligned4(r.p)) return kErrAlign;
  }
  if (!aligned4(x) || !aligned4(h) || !aligned4(out) || !aligned4(normed)) return kErrAlign;
  DeviceRanges ptrs;
  TSPLAT_CHECK(ptrs.check(x, rx.bytes()));
  TSPLAT_CHECK(ptrs.check(h, rh.bytes()));
  TSPLAT_CHECK(ptrs.check(out, ro.bytes()));
  TSPLAT_CHECK(ptrs.check(normed, rn.bytes()));
  for (const Rows& r : reads)
    if (r.p) TSPLAT_CHECK(ptrs.check(r.p, r.bytes()));
  ResidualNormParams p{x, h, out, normed, x_stride, h_stride, out_stride, normed_stride, rows, cols,
                       residual_scale, gate, gate_stride,
                       NormSpec{post_kind, post_weight, post_bias, post_eps},
                       NormSpec{pre_kind, pre_weight, pre_bias, pre_eps},
                       scale, shift, mod_stride, per};
  return launched(launch_residual_norm(p, static_cast<hipStream_t>(stream)));
}

int tsplat_rope_axes_async(const float* x, int64_t part_stride, int64_t batch_stride, int64_t token_stride,
                           int64_t head_stride, int parts, const float* gamma0, const float* gamma1,
                           float* out0, float* out1, float* out2, const void* positions, int position_type,
                           int position_batches, int axes, const double* turns, const int32_t* axis,
                           int interleaved, float eps, int B, int L, int H, int D, int out_bhld, void* stream) {
  if (!x || !out0 || !positions || !turns || !axis) return kErrNull;
  if (parts < 1 || parts > 3 || B <= 0 || L <= 0 || H <= 0 || D <= 0 || (D & 1) || D > kMaxHeadDim || H > kMaxHeads)
    return kErrDims;
  if ((parts > 1 && !out1) || (parts > 2 && !out2)) return kErrNull;
  if (axes < 1 || axes > kMaxAxes || (position_type != 0 && position_type != 1) || !(eps >= 0.0f)) return kErrDims;
  if (position_batches != 1 && position_batches != B) return kErrRange;
  const int64_t tokens = (int64_t)B * L;
  if (tokens > INT32_MAX) return kErrDims;  // (the launch's grid holds 2^32 groups of a token at least)
  const int64_t steps[4][2] = {{parts, part_stride}, {B, batch_stride}, {L, token_stride}, {H, head_stride}};
  __int128 last = D;
  for (const auto& s : steps) {
    if (s[0] > 1 && s[1] < D) return kErrRange;
    if (s[0] > 1) last += (__int128)(s[0] - 1) * s[1];
  }
  if (last > (INT64_C(1) << 58)) return kErrRange;  // (bytes stay far from the end of 64 bits)
  const int64_t in_last = (int64_t)last;
  float* outs[3] = {out0, parts > 1 ? out1 : nullptr, parts > 2 ? out2 : nullptr};
  const Rows in{x, in_last, 1, in_last};
  const int64_t values = tokens * H * D, places = position_batches * (int64_t)L * axes;
  // all that is read, in floats
  const Rows reads[] = {in, whole(gamma0, (int64_t)H * D), whole(parts > 1 ? gamma1 : nullptr, (int64_t)H * D),
                        whole(positions, places), whole(turns, D), whole(axis, D / 2)};
  if (!aligned4(x) || !aligned4(positions) || !aligned4(axis) || (reinterpret_cast<uintptr_t>(turns) & 7u) ||
      !aligned4(gamma0) || !aligned4(gamma1))
    return kErrAlign;
  for (int i = 0; i < parts; ++i) {
    const Rows o{outs[i], values, 1, values};
    if (!aligned4(outs[i])) return kErrAlign;
    for (const Rows& r : reads)
      if (r.p && !disjoint(o, r)) return kErrRange;
    for (int j = 0; j < i; ++j)
      if (!disjoint(o, Rows{outs[j], values, 1, values})) return kErrRange;
  }
  DeviceRanges ptrs;
  for (int i = 0; i < parts; ++i) TSPLAT_CHECK(ptrs.check(outs[i], values * 4));
  for (const Rows& r : reads)
    if (r.p) TSPLAT_CHECK(ptrs.check(r.p, r.bytes()));
  RopeAxesParams p{x, part_stride, batch_stride, token_stride, head_stride, parts, {gamma0, gamma1},
                   {outs[0], outs[1], outs[2]}, positions, position_type, position_batches, axes, turns, axis,
                   interleaved ? 1 : 0, eps, B, L, H, D, out_bhld ? 1 : 0};
  return launched(launch_rope_axes(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
