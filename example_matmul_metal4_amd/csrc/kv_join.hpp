// Partial sums of attention over the paged cache in few bits, and their join (kv_attention.hip, kv_prefill.hip).
#pragma once

#include "kv_device.hpp"

namespace mtk {

// Weights are exp2(score - offset). An offset is raised to the scores' maximum less kKvLift<DT> once that is more than kKvSlack
// above it, so that sums are rarely rescaled: the largest weight lies in 2^lift to 2^(lift + slack). They go to the second
// product in 16 bits; f16 holds none below 2^-25, which with a lift of 7 is 2^-32 of the row's largest (without, 2^-25: of 131072
// positions 0.4 % of the sum could be lost), while 2^15 and the rounding above stay in its range. bf16 has the range of fp32.
template <int DT>
constexpr float kKvLift = DT == DT_F16 ? 7.0f : 0.0f;
constexpr float kKvSlack = 8.0f;

// Sums of some keys of a row (4 dims), unscaled, with their exponent offset (log2) and the sum of the weights.
struct KvPart {
  float m = -INFINITY, l = 0.0f;
  f32x4 x = f32x4{};
};
__device__ __forceinline__ void add_part(KvPart &s, const KvPart &t) {
  const float m = fmaxf(s.m, t.m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  const float f = __builtin_amdgcn_exp2f(s.m - m0), g = __builtin_amdgcn_exp2f(t.m - m0);
  // an offset of -inf has no keys: its sums count as they are
  s.l = s.l * (s.m == -INFINITY ? 1.0f : f) + t.l * (t.m == -INFINITY ? 1.0f : g);
  s.x = s.x * (s.m == -INFINITY ? 1.0f : f) + t.x * (t.m == -INFINITY ? 1.0f : g);
  s.m = m;
}

// The offset that a row's sums start with: rows that see a key are told from those that see none by it, also where all their
// scores are -inf.
__device__ __forceinline__ float first_offset(bool sees) { return sees ? -3.402823466e38f : -INFINITY; }
// What a row's sums are divided by its weights' sum with. No weights: zeros where it sees no key, NaN where all its scores
// are -inf.
__device__ __forceinline__ float inverse_of(float l, float m) {
  return l != 0.0f ? 1.0f / l : m == -INFINITY ? 0.0f : __builtin_nanf("");
}

// 4 dims of (packed row, query head) from d on; the row's log-sum-exp with d == 0.
template <int DT>
__device__ __forceinline__ void store_out(const mtk_kv_attn_kargs &a, int row, int h, int d, const KvPart &s) {
  const float inv = inverse_of(s.l, s.m);
  if (d < a.D)
    *(u32x2 *)((uint16_t *)a.O + ((size_t)row * a.H + h) * a.D + d) =
        u32x2{pack2<DT>(s.x.x * inv, s.x.y * inv), pack2<DT>(s.x.z * inv, s.x.w * inv)};
  if (d == 0 && a.lse)
    a.lse[(size_t)row * a.H + h] = s.l == 0.0f ? -INFINITY : (s.m == -INFINITY ? s.l : s.m + __builtin_amdgcn_logf(s.l)) * 0.6931471805599453f;
}

// The partial sums of each (row, query head) of a pair that workgroups share, in an order that their number fixes.
// A group of D / 4 lanes (4 dims each) adds parts, kAhead of them in flight at once.
//   PARTS: a workgroup has one (row, query head); group g of NG adds every NGth part, the groups are added in turn. For
//   few pairs of long sequences, which have many parts.
//   else: each group has a query head of its own, a workgroup NG heads of a row.
// Bound by latency (the lengths, the parts' statistics and the parts in turn): 4.6 us for 128 rows of heads, 7.0 for one row
// of 32 heads in 128 parts each. runtime: plan_kv_attn has both sides of the choice.
constexpr int kKvJoin = 256;  // threads
template <int DT, bool PARTS>
__device__ __forceinline__ void kv_join(const mtk_kv_attn_kargs &a, int block, int n_blocks, int (*sm_line)[kLineWords]) {
  __shared__ f32x4 sm_x[PARTS ? kKvJoin : 1];
  __shared__ f32x2 sm_ml[PARTS ? kKvJoin : 1];
  const int tid = threadIdx.x, lane = tid & 63, G = a.G, rows = 1 << a.rows_shift;
  const int chunks = a.part_ld / 4, groups = kKvJoin / chunks;
  const int g = tid / chunks, d = 4 * (tid - g * chunks);
  const int heads = PARTS ? 1 : groups, per_row = (a.H + heads - 1) / heads;  // items of a row
  if (block >= a.T * per_row) return;
  KvLine<0, 0> line(a, lane, sm_line[tid >> 6]);
  line.lay();
  int length, base, pairs, blocks;
  KvSegment seq;
  auto open = [&](int l) {
    seq = line.sequence(l, length, base, pairs);
    blocks = kv_div(pairs, a.H_kv);
    return !(pairs == 0 || (line.cut.padded && length == line.cut.each));  // none of its pairs is shared
  };
  // Items are taken in turn by the workgroups, as the rows that are shared may lie together; uniform: every wavefront of a
  // workgroup takes the same ones.
  kv_walk(line, a.T, per_row, a.S_q, block, n_blocks, open, [&](int it) {
    const int t = it / per_row, h = (it - t * per_row) * heads + (PARTS ? 0 : g);
    const bool mine = g < groups && h < a.H;  // lanes behind the last group, or behind the last head, add nothing
    if (!PARTS && !mine) return;  // PARTS: they reach the barriers below with the others
    const int hk = kv_div(h, G), r = (t - seq.seq.first) * G + h - hk * G, rb = r >> a.rows_shift;
    const int start = base + ((a.by_pair ? blocks - 1 - rb : rb) * a.H_kv + hk) * length;
    const int w0 = kv_div(start, line.cut.each), w1 = min(kv_div(start + seq.steps - 1, line.cut.each), a.places - 1);
    if (w0 >= w1) return;  // one workgroup's
    const int first = start == w0 * line.cut.each ? 0 : 1;
    KvPart sum;
    constexpr int kAhead = 8;
    const int step = PARTS ? groups : 1;
    for (int s0 = w0 + (PARTS ? g : 0); mine && s0 <= w1; s0 += kAhead * step) {
      KvPart p[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int w = s0 + i * step;
        if (w <= w1) {
          const size_t place = a.by_pair ? (size_t)w : (size_t)w * 2 + (w == w0 ? first : 0);
          const size_t at = (place << a.rows_shift) + (r & (rows - 1));
          const f32x2 ml = *(const f32x2 *)(a.part_ml + 2 * at);
          p[i] = KvPart{ml.x, ml.y, *(const f32x4 *)(a.part + at * a.part_ld + d)};
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add_part(sum, p[i]);
    }
    if constexpr (PARTS) {
      __syncthreads();
      sm_x[tid] = sum.x;
      sm_ml[tid] = f32x2{sum.m, sum.l};
      __syncthreads();
      if (tid < chunks) {
        for (int i = 1; i < min(groups, w1 - w0 + 1); ++i) {
          const int k = tid + i * chunks;
          add_part(sum, KvPart{sm_ml[k].x, sm_ml[k].y, sm_x[k]});
        }
        store_out<DT>(a, t, h, d, sum);
      }
    } else {
      store_out<DT>(a, t, h, d, sum);
    }
  });
}

}  // namespace mtk
