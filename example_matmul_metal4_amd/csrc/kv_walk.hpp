// Which items of a join (kv_join.hpp) a workgroup takes: plain functions over a view of the batch that shows 64 sequences at a
// time, for the kernels (KvLine) and the CPU tests.
//
// A view has
//   windows()    how many windows of 64 sequences there are
//   hit(t)       the place in this window of the sequence that packed row t belongs to, or -1
//   later(t)     the first row behind t that a sequence of this window has, or INT32_MAX
//   step()       on to the next window, from the last one to the first
//   rows_of(l)   first row and rows of the sequence at place l
#pragma once

#include "kv_cache.h"

typedef struct {
  int first, rows;
} kv_rows;

// The place of row t's sequence, in the window that the view then shows. Where no sequence has row t (rows before the first one,
// behind the last), t becomes the next row that one has; none: -1. Rows are asked for in ascending order, so that the windows
// are walked once, but for rows of no sequence: those need a look at all of them, once for each gap.
template <typename View>
MTK_KV_FN int kv_find_row(View &view, int &t) {
  for (;;) {
    int next = INT32_MAX;
    for (int n = view.windows(); n > 0; --n) {
      const int l = view.hit(t);
      if (l >= 0) return l;
      const int x = view.later(t);
      next = x < next ? x : next;
      view.step();
    }
    if (next == INT32_MAX) return -1;
    t = next;
  }
}

// Of the T * per_row items (per_row for each packed row) those numbered block, block + n_blocks and so on: item(it) for each
// one whose row a sequence has, at most S_q rows of each. open(l): before a sequence's first one; false: there is nothing to do.
template <typename View, typename Open, typename Item>
MTK_KV_FN void kv_walk(View &view, int T, int per_row, int S_q, int block, int n_blocks, const Open &open, const Item &item) {
  const int items = T * per_row;
  auto past = [&](int it, int64_t end) {  // the first of this workgroup's items from `end` on
    return end > it ? it + (int)((end - it + n_blocks - 1) / n_blocks) * n_blocks : it;
  };
  for (int it = block; it < items;) {
    const int row = it / per_row;
    int t = row;
    const int l = kv_find_row(view, t);
    if (l < 0) return;
    if (t > row) {
      it = past(it, (int64_t)t * per_row);
      continue;
    }
    const kv_rows s = view.rows_of(l);
    if (open(l)) {
      const int64_t end = (int64_t)(s.first + (s.rows < S_q ? s.rows : S_q)) * per_row;
      for (; it < end; it += n_blocks) item(it);
    }
    it = past(it, (int64_t)(s.first + s.rows) * per_row);
  }
}
