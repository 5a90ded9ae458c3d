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

#endif
