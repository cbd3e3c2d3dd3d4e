// The plan of a ragged cross attention: its layout, what its header says, and the tiles that the kernels take.
#pragma once

#include <stdint.h>

namespace tsplat {

// The plan's ints: the header, then `items` work items of kCrossItem ints, then `joins` of kCrossJoin.
enum CrossHeader : int {
  kPlanMagic = 0, kPlanInts, kPlanItems, kPlanJoins, kPlanParts, kPlanRows, kPlanStates, kPlanHeads, kPlanKvHeads,
  kPlanDim, kPlanType, kPlanTerms, kPlanFew, kPlanHeaderInts = 16
};
constexpr int32_t kPlanMagicValue = 0x54435031;

// One workgroup's work for one key head: `rows` rows from row0 of a request's query rows, where a row is a query token
// and one of the group's heads (row = token * group + head), against `keys` states from key0 on.
// part: where the partial result goes, or -1: the result itself.
struct CrossItem {
  int32_t token0;  // the request's first query token
  int32_t row0, rows;
  int32_t key0, keys;
  int32_t part;
  int32_t unused[2];
};
// The same rows' partial results, `parts` of them from first_part on, become the result.
struct CrossJoin {
  int32_t token0, row0, rows, first_part, parts;
  int32_t unused[3];
};
constexpr int kCrossItem = sizeof(CrossItem) / 4, kCrossJoin = sizeof(CrossJoin) / 4;

// Head sizes are padded to one of these.
constexpr int cross_padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }

// A workgroup's tile: wq waves of 32 rows each against kb blocks of 32 states; few: 32 rows, a block of 32 states to each
// of kFewWaves waves.
constexpr int kFewWaves = 4;
struct CrossTile {
  int wq, kb;
};
constexpr CrossTile cross_tile(int padded, int terms, bool few) {
  if (few) return {1, kFewWaves};
  if (terms > 1) return {8, padded > 64 ? 1 : 2};
  return {4, 2};
}

// Whether a launch holds a workgroup for each item and key head: its threads are counted in 32 bits.
inline bool cross_launch_fits(int64_t items, int64_t kv_heads, const CrossTile& tile, bool few) {
  return items * kv_heads * ((few ? kFewWaves : tile.wq) * 64) <= UINT32_MAX;
}

// Writes the plan (null: only counts); its size in ints, or a negative status.
int64_t make_cross_plan(const int32_t* q_lengths, const int32_t* k_lengths, int requests, int heads, int kv_heads,
                        int head_dim, int dtype, int precision, int compute_units, int32_t* plan, int64_t plan_ints);

// Floats of one part and key head: the rows' sums of padded columns, then their maxima, then their denominators.
inline int64_t cross_part_floats(const int32_t* header) {
  const int padded = cross_padded_dim(header[kPlanDim]);
  return (int64_t)cross_tile(padded, header[kPlanTerms], header[kPlanFew] != 0).wq * 32 * (padded + 2);
}

// Whether a call may go by pairs of fp16 values (cross_pairs.hip): fp32 at fp32 accuracy, many rows.
inline bool cross_has_pairs(const int32_t* header) {
  return header[kPlanType] == 0 && header[kPlanTerms] == 3 && header[kPlanFew] == 0;
}

}  // namespace tsplat
