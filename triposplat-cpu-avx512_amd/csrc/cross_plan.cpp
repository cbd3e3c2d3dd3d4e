// The plan of a ragged cross attention (cross_plan.h): rows in tiles, and keys in parts where the tiles alone would not
// keep the GPU busy or where one request's keys would outlast the others.

#include "cross_plan.h"

#include <algorithm>

#include "../../include/tsplat_hip_cross.h"
#include "tsplat_common.h"

namespace tsplat {

static_assert(kPlanHeaderInts == TSPLAT_CROSS_HEADER, "the header's size is part of the interface");

int64_t make_cross_plan(const int32_t* q_lengths, const int32_t* k_lengths, int requests, int heads, int kv_heads,
                        int head_dim, int dtype, int precision, int compute_units, int32_t* plan, int64_t plan_ints) {
  if (requests < 0 || requests > (1 << 20) || heads < 1 || heads >= (1 << 16) || kv_heads < 1 || heads % kv_heads != 0 ||
      head_dim < 1 || head_dim > 128 || dtype < 0 || dtype > 2 || precision < 0 || precision > 2 ||
      (dtype != 0 && precision != 0))
    return kErrDims;
  if (requests > 0 && (!q_lengths || !k_lengths)) return kErrNull;
  const int group = heads / kv_heads;
  int64_t rows_all = 0, states_all = 0, longest = 0;
  for (int i = 0; i < requests; ++i) {
    if (q_lengths[i] < 0 || k_lengths[i] < 0) return kErrDims;
    rows_all += q_lengths[i], states_all += k_lengths[i];
    longest = std::max<int64_t>(longest, (int64_t)q_lengths[i] * group);
  }
  if (rows_all * group > INT32_MAX / 2 || states_all > INT32_MAX / 2) return kErrDims;
  const int padded = cross_padded_dim(head_dim);
  const int terms = dtype != 0 ? 1 : precision == 0 ? 3 : precision;
  const bool few = longest <= 32;
  const CrossTile tile = cross_tile(padded, terms, few);
  const int tile_rows = tile.wq * 32, tile_keys = tile.kb * 32;
  // Tiles of keys over all workgroups: an even share of them for each workgroup that runs at once is the length of a part
  // (four times as many parts for few rows, whose sums are small).  Where that is short, the length that makes one part's
  // tiles, in a chain, and the join of a request's parts together shortest: their number halved, its root.  (Two single
  // tokens over 2049 and 4101 states in fp32: parts of 1, 2, 3, 4 tiles take 34, 27, 26, 23 us; one over 500: 9.9, 11.5,
  // 11.5, 14; 64 over 4096: 2, 3, 4, 6 take 38, 37, 26, 26; three of 200 over 700 in 16 bits: 2, 3, 4 take 14.1, 12.4, 12.5.)
  // The even share counts one workgroup of eight waves a CU (fp32, 2000 rows over 2000 states, 16 heads: 69 us, for two at
  // once 83), which is what fits, and two of four waves (16 bits, five ragged requests of 1 to 8193 rows: 92, for one 105),
  // of which three fit for heads up to 64 and two for wider ones.
  const int64_t at_once = (int64_t)compute_units * (few ? 8 : terms > 1 ? 1 : 2);
  int64_t work = 0, most = 0;
  for (int i = 0; i < requests; ++i) {
    const int64_t tiles = (k_lengths[i] + (int64_t)tile_keys - 1) / tile_keys;
    work += ((int64_t)q_lengths[i] * group + tile_rows - 1) / tile_rows * tiles;
    if (q_lengths[i] > 0) most = std::max(most, tiles);
  }
  int64_t share = few ? 1 : terms > 1 ? 2 : 3;
  while ((share + 1) * (share + 1) * 2 <= most) ++share;
  share = std::max<int64_t>(share, (work * kv_heads + at_once - 1) / at_once);

  int64_t items = 0, joins = 0, parts = 0;
  const int64_t room_items = plan ? (plan_ints - kPlanHeaderInts) / kCrossItem : 0;
  CrossItem* item = plan ? reinterpret_cast<CrossItem*>(plan + kPlanHeaderInts) : nullptr;
  auto each = [&](auto emit_item, auto emit_join) {
    int32_t token0 = 0, key0 = 0;
    for (int i = 0; i < requests; ++i) {
      const int32_t rows = q_lengths[i] * group, keys = k_lengths[i];
      const int64_t tiles = ((int64_t)keys + tile_keys - 1) / tile_keys;
      const int32_t n = (int32_t)std::max<int64_t>(1, (tiles + share - 1) / share);
      for (int32_t row0 = 0; row0 < rows; row0 += tile_rows) {
        const int32_t live = std::min(tile_rows, rows - row0);
        if (n > 1) emit_join(CrossJoin{token0, row0, live, (int32_t)parts, n, {0, 0, 0}});
        for (int32_t p = 0; p < n; ++p) {
          const int32_t from = (int32_t)(tiles * p / n) * tile_keys;
          const int32_t to = std::min<int32_t>(keys, (int32_t)(tiles * (p + 1) / n) * tile_keys);
          emit_item(CrossItem{token0, row0, live, key0 + from, to - from, n > 1 ? (int32_t)parts++ : -1, {0, 0}});
        }
      }
      token0 += q_lengths[i], key0 += keys;
    }
  };
  each([&](const CrossItem&) { ++items; }, [&](const CrossJoin&) { ++joins; });
  const int64_t need = kPlanHeaderInts + items * kCrossItem + joins * kCrossJoin;
  if (!cross_launch_fits(items, kv_heads, tile, few) || need > INT32_MAX) return kErrDims;
  if (!plan) return need;
  if (plan_ints < need || room_items < items) return kErrRange;
  const int32_t header[kPlanHeaderInts] = {kPlanMagicValue, (int32_t)need, (int32_t)items, (int32_t)joins,
                                           (int32_t)parts, (int32_t)rows_all, (int32_t)states_all, heads, kv_heads,
                                           head_dim, dtype, terms, few ? 1 : 0, 0, 0, 0};
  std::copy(header, header + kPlanHeaderInts, plan);
  CrossJoin* join = reinterpret_cast<CrossJoin*>(plan + kPlanHeaderInts + items * kCrossItem);
  parts = 0;
  CrossItem* const first = item;
  each([&](const CrossItem& it) { *item++ = it; }, [&](const CrossJoin& j) { *join++ = j; });
  // the longest first: what starts last is short
  std::sort(first, item, [](const CrossItem& a, const CrossItem& b) {
    if (a.keys != b.keys) return a.keys > b.keys;
    return a.key0 != b.key0 ? a.key0 < b.key0 : a.token0 != b.token0 ? a.token0 < b.token0 : a.row0 < b.row0;
  });
  return need;
}

}  // namespace tsplat
