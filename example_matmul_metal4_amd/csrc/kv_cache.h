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

/* Rows of a wavefront that writes or reads rows, at most: the loads of all of them are in flight at once. */
enum { KV_MOVE_ROWS = 4 };

// One sequence of the batch, from its entries of row_start and kv_len, whatever they hold. Its rows are
// [first, first + rows) of the packed tensors, row i at position pos0 + i. len: kv_len; keys: cached positions, at most
// the table's; bad: kv_len is more than the table holds.
typedef struct {
  int first, rows, len;
  int64_t pos0;
  int keys, bad;
} kv_seq;

MTK_KV_FN kv_seq kv_sequence(int start, int next, int len, int T, int max_pages, int page_shift) {
  kv_seq s;
  const int cap = max_pages << page_shift;
  s.first = start < 0 ? 0 : start > T ? T : start;
  const int last = next < s.first ? s.first : next > T ? T : next;
  s.rows = last - s.first;
  s.len = len;
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

// x / d for 0 <= x < 2^31, 0 < d <= 2^24.
MTK_KV_FN int kv_div(int x, int d) {
#ifdef __HIP_DEVICE_COMPILE__
  // by a reciprocal in 32 bits: at most x 2^-22 / d + 1 off, so a second estimate of the rest is at most one off
  const float inv = __builtin_amdgcn_rcpf((float)d);
  int q = (int)((float)x * inv);
  int r = (int)((uint32_t)x - (uint32_t)q * (uint32_t)d);
  const int e = (int)((float)r * inv);
  q += e;
  r -= e * d;
  return q + (r < 0 ? -1 : r >= d ? 1 : 0);
#else
  return x / d;
#endif
}

// Who does what in attention. A sequence has `blocks` blocks of 2^rows_shift (row, query head) pairs for each K/V head,
// and `steps` steps of 2^step_shift keys (at least one). The (block, head) pairs of all sequences, one sequence after another,
// lie on a line; workgroup w has the steps from w * each to (w + 1) * each of it, so that all of them have the same work, whatever
// the lengths. A pair that a boundary cuts leaves partial sums.
//   each = max(least, work / units), so that there are at most `units` workgroups.
// Where so little work is left that pairs of their own workgroups (ceil(steps / least) each) are no more than `units`,
// a pair's length on the line is rounded up to a multiple of `each` = least: no workgroup has parts of two pairs.
typedef struct {
  int blocks, steps;
} kv_share;

MTK_KV_FN kv_share kv_blocks(kv_seq s, int S_q, int G, int rows_shift, int step_shift, int rows_above, int rows_most) {
  kv_share r;
  const uint32_t pairs = (uint32_t)(s.rows < S_q ? s.rows : S_q) * (uint32_t)G;  // S_q * G < 2^31
  const int mine = pairs > (uint32_t)rows_above && pairs <= (uint32_t)rows_most;
  r.blocks = mine ? (int)((pairs + (1u << rows_shift) - 1) >> rows_shift) : 0;
  r.steps = (int)(((uint32_t)s.keys + (1u << step_shift) - 1) >> step_shift);
  if (r.steps < 1) r.steps = 1;
  return r;
}

// Workgroups of a pair's own, of `least` steps each.
MTK_KV_FN int kv_own(kv_share r, int least) { return kv_div(r.steps + least - 1, least); }

typedef struct {
  int each;   /* steps of a workgroup */
  int padded; /* a pair's length is a multiple of it */
} kv_cut;

// From the sums over all sequences of blocks * heads * steps and blocks * heads * kv_own.
MTK_KV_FN kv_cut kv_cut_of(int work, int own, int units, int least) {
  kv_cut c;
  c.padded = own <= units;
  c.each = least;
  if (!c.padded) {
    const int n = kv_div(work + units - 1, units);
    if (n > least) c.each = n;
  }
  return c;
}

// Launches whose workgroups have one pair each (by_pair). own: the pairs. Whether they have more than one workgroup each: not
// where they are `units` or more, nor where two shares of one, of `few` steps or less on average, gain less than the join costs
// (32 heads, 8 K/V heads of 128 dims, 500 rows in 2 sequences each: 16 steps of 64 keys 38.1 us whole, 47.2 in two shares; 24 steps
// 49.7 and 54.1; 32 steps 61.1 and 61.2; 200 rows in 4: 39.3 and 45.7, 51.1 and 52.6, 62.9 and 59.1).
#define KV_FEW_STEPS 28 /* of 64 keys */
MTK_KV_FN int kv_few_steps(int step_shift) { return (KV_FEW_STEPS << 6) >> step_shift; }
MTK_KV_FN int kv_pairs_split(int work, int own, int units, int few = KV_FEW_STEPS) {
  return own < units && (own <= units / 3 || work > few * own);
}

// Steps of a share, at least `least` and no more than `most`, the steps of a full table. With this or more there are at most
// `units` workgroups: pairs ceil their steps / each, which adds less than 1 for each.
MTK_KV_FN int kv_each_of_pairs(int work, int own, int units, int least, int most, int few = KV_FEW_STEPS) {
  int each = kv_pairs_split(work, own, units, few) ? kv_div(work + (units - own) - 1, units - own) : most;
  if (each > most) each = most;
  return each < least ? least : each;
}

// The steps of such a launch, 2^shift keys each: 64, but more where the sums over `pairs` pairs of full tables would not fit 32
// bits (a pair's padded length and a share past it). `pairs` counts S_q rows of every sequence, as no less is sure whatever
// row_start holds; starts that ascend make far fewer, whose shares are then just longer. least: shares of 256 keys or more where
// pairs may be split, else whole ones.
typedef struct {
  int shift; /* -1: none fits */
  int steps, least;
} kv_pair_steps;
MTK_KV_FN kv_pair_steps kv_steps_of_pairs(int64_t pairs, int64_t positions, int split) {
  kv_pair_steps s;
  for (s.shift = 6; s.shift <= 30; ++s.shift) {
    s.steps = (int)((positions + ((int64_t)1 << s.shift) - 1) >> s.shift);
    s.least = split ? (s.shift < 8 ? 256 >> s.shift : 1) : s.steps;
    if (pairs <= INT32_MAX / (3 * (int64_t)s.steps + s.least)) return s;
  }
  s.shift = -1;
  return s;
}

MTK_KV_FN int kv_length(kv_share r, kv_cut c) { return c.padded ? kv_div(r.steps + c.each - 1, c.each) * c.each : r.steps; }

// Most row blocks per K/V head of a launch.
MTK_KV_FN int64_t kv_max_blocks(int B, int T, int S_q, int G, int rows) {
  const int64_t each = (int64_t)B * (((int64_t)S_q * G + rows - 1) / rows);
  const int64_t all = (int64_t)T * G / rows + B;
  return each < all ? each : all;
}

#endif
