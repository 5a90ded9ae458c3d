// Layout of the paged key/value cache in few bits, and which workgroup of an attention launch does what:
// plain functions that the host runtime, the kernels and the CPU tests share.
//
// A page holds 2^page_shift positions. The region of (page, K/V head) is [K codes][V codes][K scales][V scales],
// codes [position][blocks][16 or 32 bytes], scales [position][blocks]; regions lie [page][head]. Block: 32 dims
// of one position and head (dims past D are zeros). fp4: e2m1, two codes per byte, the even dim in the low half;
// fp8: e4m3. A scale byte s stands for 2^(s - 127); 255: the block is NaN.
#ifndef MTK_KV_CACHE_H
#define MTK_KV_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define MTK_KV_FN static __host__ __device__ __forceinline__
#else
#define MTK_KV_FN static inline
#endif

enum { KV_FP4 = 0, KV_FP8 = 1 };

MTK_KV_FN int kv_row_bytes(int fmt, int blocks) { return blocks * (fmt == KV_FP4 ? 16 : 32); }

// Bytes of the region of a page and head.
MTK_KV_FN uint64_t kv_region_bytes(int fmt, int blocks, int page_shift) {
  return ((uint64_t)2 * (uint64_t)(kv_row_bytes(fmt, blocks) + blocks)) << page_shift;
}

// One sequence of the batch, from its entries of row_start and kv_len, whatever they hold. Its rows are
// [first, first + rows) of the packed tensors, row i at position pos0 + i. keys: cached positions, at most the
// table's; bad: kv_len is more than the table holds.
typedef struct {
  int first, rows;
  int64_t pos0;
  int keys, bad;
} kv_seq;

MTK_KV_FN kv_seq kv_sequence(int start, int next, int len, int T, int max_pages, int page_shift) {
  kv_seq s;
  const int cap = max_pages << page_shift;
  s.first = start < 0 ? 0 : start > T ? T : start;
  const int last = next < s.first ? s.first : next > T ? T : next;
  s.rows = last - s.first;
  s.pos0 = (int64_t)len - s.rows;
  s.bad = len > cap;
  s.keys = len < 0 ? 0 : len > cap ? cap : len;
  return s;
}

// The page of a position: a table entry in range, or -1.
MTK_KV_FN int kv_page(const int32_t *row_of_table, int64_t pos, int n_pages, int max_pages, int page_shift) {
  if (pos < 0 || (pos >> page_shift) >= max_pages) return -1;
  const int page = row_of_table[pos >> page_shift];
  return page >= 0 && page < n_pages ? page : -1;
}

// Key splits. A sequence has blocks of `rows` (row, query head) pairs of a K/V head and ceil(keys / step) steps
// of keys; one workgroup takes at most c steps of one block and head. c is the least (from `least` on) that keeps
// the launch at about `units` workgroups: work / units, then raised while the rounding up of short sequences
// still adds too many (which is looked at for up to 64 sequences).
typedef struct {
  int blocks; /* row blocks */
  int steps;
  int splits, per; /* workgroups per block and head, steps of each */
} kv_share;

MTK_KV_FN kv_share kv_blocks(kv_seq s, int S_q, int G, int rows, int step, int rows_above, int rows_most) {
  kv_share r;
  const int64_t pairs = (int64_t)(s.rows < S_q ? s.rows : S_q) * G;
  const int mine = pairs > rows_above && pairs <= rows_most;
  r.blocks = mine ? (int)((pairs + rows - 1) / rows) : 0;
  r.steps = (int)(((int64_t)s.keys + step - 1) / step);
  r.splits = 1;
  r.per = r.steps;
  return r;
}

MTK_KV_FN void kv_split(kv_share *r, int c) {
  if (r->steps <= c) {
    r->splits = 1;
    r->per = r->steps;
    return;
  }
  const int n = (r->steps + c - 1) / c;
  r->per = (r->steps + n - 1) / n;
  r->splits = (r->steps + r->per - 1) / r->per;
}

// The next c to try when `total` workgroups came out.
MTK_KV_FN int kv_next_c(int c, int total, int units) {
  const int64_t n = (int64_t)c * total / (units > 0 ? units : 1);
  return n > c ? (n < (1 << 30) ? (int)n : (1 << 30)) : c + 1;
}

// Most workgroups of a launch with these limits: each row block and head rounds its splits up by less than one.
MTK_KV_FN int64_t kv_max_blocks(int B, int T, int S_q, int G, int rows) {
  const int64_t each = (int64_t)B * (((int64_t)S_q * G + rows - 1) / rows);
  const int64_t all = (int64_t)T * G / rows + B;
  return each < all ? each : all;
}

#endif
