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

// Where the i-th tile of workgroup `block` of a grid of `grid` is among all `total`, or -1: the XCDs have contiguous runs of them (a
// workgroup is on XCD block % 8), through which the workgroups of each go in step.
MTK_GROUP_FN int group_nth_tile(int block, int grid, int i, int total) {
  const int x = block & 7, each = (grid - x + 7) >> 3;
  const int q = total >> 3, r = total & 7;
  const int at = (block >> 3) + i * each;
  return at < q + (x < r ? 1 : 0) ? (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + at : -1;
}

#endif
