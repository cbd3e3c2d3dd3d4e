// C-ABI of the ragged cross attention (include/tsplat_hip_cross.h): the plan, argument checks and extents, then the
// launches on the caller's stream.  Nothing here allocates or waits.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "capi_spans.h"
#include "cross_attention.h"
#include "../../include/tsplat_hip_cross.h"

using namespace tsplat;

namespace {

constexpr int kCrossAbiVersion = 1;
constexpr float kLog2e = 1.4426950408889634f;  // (the kernels' exponents are base 2)

int launched(int st) {
  if (st == kErrLaunch) (void)note(hipErrorLaunchFailure);
  return st;
}

// Vectors of `dim` values at [token][head]: rows of the outer of the two strides.
struct Vectors {
  bool sane;
  Span span;
};
Vectors vectors(const void* p, int64_t token, int64_t head, int64_t tokens, int64_t heads, int64_t dim, int size) {
  int64_t outer = token, inner = head, outers = tokens, inners = heads;
  if (outers > 1 && inners > 1 && outer < inner) outer = head, inner = token, outers = heads, inners = tokens;
  if (outers == 1) outer = inner, outers = inners, inners = 1;
  if (!sane_rows(inner, inners, dim)) return {false, {}};
  const int64_t row = inners == 1 ? dim : (inners - 1) * inner + dim;
  if (!sane_rows(outer, outers, row)) return {false, {}};
  return {true, span_rows(p, outer, outers, row, size)};
}

// Whether this is a header that tsplat_cross_plan wrote, as far as its own numbers tell.
bool is_header(const int32_t* h) {
  if (h[kPlanMagic] != kPlanMagicValue) return false;
  const int64_t ints = kPlanHeaderInts + (int64_t)h[kPlanItems] * kCrossItem + (int64_t)h[kPlanJoins] * kCrossJoin;
  return h[kPlanItems] >= 0 && h[kPlanJoins] >= 0 && h[kPlanParts] >= 0 && h[kPlanParts] <= h[kPlanItems] &&
         h[kPlanJoins] <= h[kPlanParts] && h[kPlanInts] == ints && h[kPlanRows] >= 0 && h[kPlanStates] >= 0 &&
         h[kPlanKvHeads] >= 1 && h[kPlanHeads] >= h[kPlanKvHeads] && h[kPlanHeads] % h[kPlanKvHeads] == 0 &&
         h[kPlanHeads] < 1 << 16 && h[kPlanDim] >= 1 && h[kPlanDim] <= 128 && h[kPlanType] >= 0 && h[kPlanType] <= 2 &&
         h[kPlanTerms] >= 1 && h[kPlanTerms] <= 3 && (h[kPlanType] == 0 || h[kPlanTerms] == 1) &&
         (h[kPlanFew] == 0 || h[kPlanFew] == 1) &&
         cross_launch_fits(h[kPlanItems], h[kPlanKvHeads],
                           cross_tile(cross_padded_dim(h[kPlanDim]), h[kPlanTerms], h[kPlanFew] != 0), h[kPlanFew] != 0);
}

// The parts' sums, then the pairs' flags.
int64_t part_bytes(const int32_t* h) { return (int64_t)h[kPlanParts] * h[kPlanKvHeads] * cross_part_floats(h) * 4; }
int64_t scratch_bytes(const int32_t* h) {
  return part_bytes(h) + (cross_has_pairs(h) ? ((int64_t)h[kPlanItems] * h[kPlanKvHeads] * 4 + 15) / 16 * 16 : 0);
}

bool multiple(int64_t stride, int64_t count, int of) { return count == 1 || stride % of == 0; }

}  // namespace

extern "C" {

int tsplat_cross_abi_version(void) { return kCrossAbiVersion; }

int64_t tsplat_cross_plan(const int32_t* q_lengths, const int32_t* k_lengths, int requests, int heads, int kv_heads,
                          int head_dim, int dtype, int precision, int32_t* plan, int64_t plan_ints) {
  return make_cross_plan(q_lengths, k_lengths, requests, heads, kv_heads, head_dim, dtype, precision, compute_units(),
                         plan, plan_ints);
}

int64_t tsplat_cross_scratch_bytes(const int32_t* header) {
  return header && is_header(header) ? scratch_bytes(header) : 0;
}

int tsplat_cross_attention_async(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                                 int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const float* bias,
                                 float scale, void* out, int64_t out_token, int64_t out_head, const int32_t* header,
                                 const int32_t* plan, void* scratch, int64_t scratch_size, void* stream) {
  if (!header) return kErrNull;
  if (!is_header(header) || !(scale > 0.0f) || !std::isfinite(scale * kLog2e)) return kErrDims;
  const int32_t* h = header;
  const int64_t rows = h[kPlanRows], states = h[kPlanStates];
  const int heads = h[kPlanHeads], kv_heads = h[kPlanKvHeads], dim = h[kPlanDim], size = h[kPlanType] == 0 ? 4 : 2;
  if (rows == 0) return kOk;
  if (!q || !out || !plan || (states > 0 && (!k || !v))) return kErrNull;
  const Vectors vq = vectors(q, q_token, q_head, rows, heads, dim, size);
  const Vectors vo = vectors(out, out_token, out_head, rows, heads, dim, size);
  if (!vq.sane || !vo.sane) return kErrRange;
  Span reads[5] = {vq.span, span_whole(plan, (int64_t)h[kPlanInts] * 4), {}, {}, {}};
  int count = 2;
  if (states > 0) {
    const Vectors vk = vectors(k, k_token, k_head, states, kv_heads, dim, size);
    const Vectors vv = vectors(v, v_token, v_head, states, kv_heads, dim, size);
    if (!vk.sane || !vv.sane) return kErrRange;
    reads[count++] = vk.span, reads[count++] = vv.span;
    if (bias) reads[count++] = span_whole(bias, states * 4);
  } else {
    bias = nullptr;
  }
  const int64_t need = scratch_bytes(h);
  if (need > 0 && (scratch == nullptr || scratch_size < need)) return kErrWorkspace;
  const Span room = span_whole(need > 0 ? scratch : nullptr, need);
  for (int i = 0; i < count; ++i)
    if (!apart(vo.span, reads[i]) || (room.p && !apart(room, reads[i]))) return kErrRange;
  if (room.p && !apart(room, vo.span)) return kErrRange;
  if (!aligned_to(q, size) || !aligned_to(out, size) || !aligned_to(bias, 4) || !aligned_to(plan, 4) ||
      (room.p && !aligned16(scratch)) || (states > 0 && (!aligned_to(k, size) || !aligned_to(v, size))))
    return kErrAlign;
  DeviceRanges ptrs;
  TSPLAT_CHECK(ptrs.check(out, vo.span.bytes()));
  for (int i = 0; i < count; ++i) TSPLAT_CHECK(ptrs.check(reads[i].p, reads[i].bytes()));
  if (room.p) TSPLAT_CHECK(ptrs.check(scratch, need));

  CrossParams p{};
  p.q = q, p.k = k, p.v = v, p.out = out, p.bias = bias, p.scale = scale;
  p.q_token = q_token, p.q_head = q_head, p.k_token = k_token, p.k_head = k_head;
  p.v_token = v_token, p.v_head = v_head, p.out_token = out_token, p.out_head = out_head;
  if (rows == 1) p.q_token = p.out_token = 0;
  if (heads == 1) p.q_head = p.out_head = 0;
  if (states == 1) p.k_token = p.v_token = 0;
  if (kv_heads == 1) p.k_head = p.v_head = 0;
  p.heads = heads, p.kv_heads = kv_heads, p.group = heads / kv_heads, p.dim = dim;
  p.type = h[kPlanType], p.terms = h[kPlanTerms], p.few = h[kPlanFew];
  p.items = reinterpret_cast<const CrossItem*>(plan + kPlanHeaderInts);
  p.joins = reinterpret_cast<const CrossJoin*>(plan + kPlanHeaderInts + (int64_t)h[kPlanItems] * kCrossItem);
  p.item_count = h[kPlanItems], p.join_count = h[kPlanJoins], p.parts = h[kPlanParts];
  p.partial = static_cast<float*>(scratch);
  const int eights = 16 / size;  // values of 16 bytes
  p.vec = dim % 8 == 0 && aligned16(q) && multiple(q_token, rows, eights) && multiple(q_head, heads, eights) &&
          aligned16(out) && multiple(out_token, rows, eights) && multiple(out_head, heads, eights) &&
          (states == 0 || (aligned16(k) && aligned16(v) && multiple(k_token, states, eights) &&
                           multiple(k_head, kv_heads, eights) && multiple(v_token, states, eights) &&
                           multiple(v_head, kv_heads, eights)));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (cross_has_pairs(h) && p.vec) {
    p.flags = reinterpret_cast<int32_t*>(static_cast<char*>(scratch) + part_bytes(h));
    const int st = launch_cross_pairs(p, s);
    if (st != kOk) return launched(st);
  }
  const int st = p.type != 0 ? launch_cross_16(p, s) : p.terms == 3 ? launch_cross_f32(p, s) : launch_cross_f32_fast(p, s);
  if (st != kOk || p.join_count == 0) return launched(st);
  return launched(launch_cross_join(p, s));
}

}  // extern "C"
