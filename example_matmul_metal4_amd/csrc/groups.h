// Rows of a packed tensor sorted by group (the experts of a layer): plain functions that the host runtime, the kernels and
// the CPU tests share.
#ifndef MTK_GROUPS_H
#define MTK_GROUPS_H

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

#define MTK_GROUP_FN static __host__ __device__ __forceinline__
#else
#define MTK_GROUP_FN static inline
#endif

typedef struct {
  int first, rows;
} group_rows;

// Group e's rows from row_start[e] and row_start[e + 1], whatever they hold: within [0, T], none where the end lies before the
// start.
MTK_GROUP_FN group_rows group_of(int start, int next, int T) {
  group_rows g;
  g.first = start < 0 ? 0 : start > T ? T : start;
  const int last = next < g.first ? g.first : next > T ? T : next;
  g.rows = last - g.first;
  return g;
}

// Blocks of `block` rows that E ascending groups of T rows in all have at most: each group with a row has one that may not be
// full.
MTK_GROUP_FN int64_t group_max_blocks(int E, int T, int block) { return (int64_t)T / block + (E < T ? E : T); }

// A workgroup's i-th tile among `total`: -1 none; half 0: all of it, 1 and 2: its upper and lower half.
//
// All workgroups of a persistent grid go through the tiles in step, `grid` of them at a time, so that tiles that take longer (a large
// group's gradients) are everybody's; of each `grid` tiles an XCD has neighbours (a workgroup is on XCD block % 8). The last round's
// tiles are spread over the XCDs, and where they are half of the grid or fewer two workgroups share each, if the tile can be halved.
typedef struct {
  int tile, half;
} group_place;

MTK_GROUP_FN group_place group_nth_tile(int block, int grid, int i, int total, int halves) {
  group_place p = {-1, 0};
  const int64_t done = (int64_t)i * grid, left = total - done;
  const int two = halves && 2 * left <= grid;
  const int n = left >= grid ? grid : left > 0 ? (int)left << two : 0;  // of this round
  const int x = block & 7, j = block >> 3, q = n >> 3, r = n & 7;
  if (j >= q + (x < r ? 1 : 0)) return p;
  const int at = x * q + (x < r ? x : r) + j;
  p.tile = (int)done + (two ? at >> 1 : at);
  p.half = two ? 1 + (at & 1) : 0;
  return p;
}

// K-tile k of `full` whole ones, taken from tile `turn` on; those behind them stay in their places.
MTK_GROUP_FN int group_turned(int k, int turn, int full) {
  if (k >= full) return k;
  k += turn;
  return k >= full ? k - full : k;
}
// Where the tiles of `place` (one of eight) start.
MTK_GROUP_FN int group_turn(int place, int full) { return (int)((int64_t)(place & 7) * full >> 3); }
// Where tiles start: 2^log_parts parts of a group's columns start apart, and a column block is 1 / 65536 of `per_block` parts wide.
typedef struct {
  int32_t on, log_parts, per_block;
} group_turns;
MTK_GROUP_FN group_turns group_turns_of(int log_parts, int across) {
  const group_turns t = {1, log_parts, (65536 << log_parts) / across};
  return t;
}
// The place of group e's tiles that have column block n. Nothing of it depends on how many rows any group has, so a row's sums have one
// order wherever its tile lies. Groups that follow each other start far apart, and so do those that are eight apart, whose weights
// may lie a power of two apart as their rows do.
MTK_GROUP_FN int group_turn_place(int e, int n, group_turns t) {
  return 5 * e + 3 * (e >> 3) + ((n * t.per_block >> 16) << (3 - t.log_parts));
}

#endif
