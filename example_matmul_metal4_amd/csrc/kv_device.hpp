// Device helpers of the kernels on the paged cache in few bits (kv_cache.h): conversions of codes, sums over a
// wavefront, and the search for a workgroup's share of the batch.
#pragma once

#include "device.hpp"
#include "kv_cache.h"
#include "kv_walk.hpp"

namespace mtk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

constexpr int kNanScale = 255;

__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Codes -> 16-bit values times the scale, two per instruction. Exact where the result is a normal number (e2m1
// and e4m3 have 2 and 4 significant bits).
template <int DT, int SEL>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {  // the codes of byte SEL
  if constexpr (DT == DT_F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
template <int DT, bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float scale) {  // the codes of a half
  if constexpr (DT == DT_F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// Words of 8 codes, and 8 values from them.
template <int FMT>
constexpr int kWords8 = FMT == KV_FP4 ? 1 : 2;
template <int DT, int FMT>
__device__ __forceinline__ u32x4 values8(const uint32_t *w, float scale) {
  if constexpr (FMT == KV_FP4)
    return u32x4{fp4_pair<DT, 0>(w[0], scale), fp4_pair<DT, 1>(w[0], scale), fp4_pair<DT, 2>(w[0], scale),
                 fp4_pair<DT, 3>(w[0], scale)};
  else
    return u32x4{fp8_pair<DT, false>(w[0], scale), fp8_pair<DT, true>(w[0], scale), fp8_pair<DT, false>(w[1], scale),
                 fp8_pair<DT, true>(w[1], scale)};
}

// Inclusive sum over the lanes up to this one (data-parallel moves within rows of 16, then across rows).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Minimum over the lanes.
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) x = min(x, __shfl_xor(x, i));
  return __builtin_amdgcn_readfirstlane(x);
}

template <typename A>
__device__ __forceinline__ kv_seq load_seq(const A &a, int b) {
  if (b >= a.B) return kv_sequence(0, 0, 0, 0, a.max_pages, a.page_shift);
  return kv_sequence(a.row_start[b], a.row_start[b + 1], a.kv_len[b], a.T, a.max_pages, a.page_shift);
}

// Some steps of one pair (kv_cache.h).
struct KvSegment {
  int b = -1;       // sequence, -1: none
  int hk, rb;       // K/V head, row block
  int from, to;     // steps
  int steps;        // of the pair
  int start;        // the pair's place on the line
  kv_seq seq;
};

// A wavefront's view of the line: 64 sequences at a time, in LDS words of its own (registers are what the kernel is
// short of). ROWS rows per block (128: the kernel whose workgroups have one pair each), STEP keys per step (0: as the
// launch says).
constexpr int kLineWords = 4 * 64;
template <int ROWS, int STEP>
struct KvLine {
  const mtk_kv_attn_kargs &a;
  const int lane;
  int *const sm;  // [4][64]: where the sequence's pairs end, first row, rows, length
  kv_cut cut{};
  int total = 0;          // length of the line
  int b0 = 0, before = 0; // the first of the 64, and where its pairs start

  __device__ __forceinline__ bool by_pair() const { return ROWS ? ROWS == 128 : a.by_pair != 0; }
  __device__ __forceinline__ kv_share share_of(const kv_seq &x) const {
    return kv_blocks(x, a.S_q, a.G, ROWS ? __builtin_ctz(ROWS ? ROWS : 1) : a.rows_shift, STEP ? __builtin_ctz(STEP ? STEP : 1) : a.step_shift,
                     a.rows_above, a.rows_most);
  }
  __device__ __forceinline__ void place(const kv_seq &s, const kv_share &h) {
    sm[lane] = before + wave_scan(h.blocks * a.H_kv * kv_length(h, cut));
    sm[64 + lane] = s.first;
    sm[128 + lane] = s.rows;
    sm[192 + lane] = s.len;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __device__ __forceinline__ KvLine(const mtk_kv_attn_kargs &args, int lane_, int *words) : a(args), lane(lane_), sm(words) {}
  __device__ __forceinline__ void lay() {
    const kv_seq s = load_seq(a, lane);
    const kv_share h = share_of(s);
    auto own_of = [&](const kv_share &x) { return x.blocks * a.H_kv * (by_pair() ? 1 : kv_own(x, a.least)); };
    int work = h.blocks * a.H_kv * h.steps, own = own_of(h);
#pragma unroll 1
    for (int b = 64; b < a.B; b += 64) {
      const kv_share x = share_of(load_seq(a, b + lane));
      work += x.blocks * a.H_kv * x.steps;
      own += own_of(x);
    }
    auto sum = [](int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); };
    work = sum(work);
    own = sum(own);
    if (by_pair()) {
      const int shift = STEP ? __builtin_ctz(STEP ? STEP : 1) : a.step_shift;
      const int most = (int)((((uint32_t)a.max_pages << a.page_shift) + (1u << shift) - 1) >> shift);
      const int few = kv_few_steps(shift);
      int hi = kv_each_of_pairs(work, own, a.units, a.least, most, few);
      if (a.B <= 64 && kv_pairs_split(work, own, a.units, few)) {  // the least that makes no more workgroups than that
        int lo = min(hi, max(a.least, kv_div(work + a.units - 1, a.units)));
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sum(h.blocks * a.H_kv * kv_div(h.steps + mid - 1, mid)) <= a.units)
            hi = mid;
          else
            lo = mid + 1;
        }
      }
      cut.padded = 1;
      cut.each = __builtin_amdgcn_readfirstlane(hi);
      place(s, h);
      return;
    }
    cut = kv_cut_of(work, own, a.units, a.least);
    cut.each = __builtin_amdgcn_readfirstlane(cut.each);
    total = cut.padded ? own * a.least : work;
    place(s, h);
  }
  __device__ __forceinline__ void show(int first, int starts) {  // the 64 sequences from `first` on, whose pairs start there
    b0 = first;
    before = starts;
    const kv_seq s = load_seq(a, b0 + lane);
    place(s, share_of(s));
  }
  __device__ __forceinline__ void next() { show(b0 + 64, __builtin_amdgcn_readfirstlane(sm[63])); }
  // The lane of the sequence that pos falls into, or -1. pos ascends from call to call.
  __device__ __forceinline__ int find(int pos) {
    for (;;) {
      const uint64_t in = __ballot(sm[lane] > pos);
      if (in) return __builtin_amdgcn_readfirstlane(__builtin_ctzll(in));
      if (b0 + 64 >= a.B) return -1;
      next();
    }
  }
  // ---- as a view of kv_walk
  __device__ __forceinline__ int windows() const { return (a.B + 63) >> 6; }
  __device__ __forceinline__ int hit(int t) const {
    const int first = sm[64 + lane];
    const uint64_t in = __ballot(b0 + lane < a.B && first <= t && t < first + sm[128 + lane]);
    return in ? __builtin_amdgcn_readfirstlane(__builtin_ctzll(in)) : -1;
  }
  __device__ __forceinline__ int later(int t) const {
    const int first = sm[64 + lane];
    return wave_min(b0 + lane < a.B && first > t && sm[128 + lane] > 0 ? first : INT32_MAX);
  }
  __device__ __forceinline__ void step() {
    if (b0 + 64 < a.B)
      next();
    else if (b0 > 0)
      show(0, 0);
  }
  __device__ __forceinline__ kv_rows rows_of(int l) const {
    return kv_rows{__builtin_amdgcn_readfirstlane(sm[64 + l]), __builtin_amdgcn_readfirstlane(sm[128 + l])};
  }
  // That sequence; the length of its pairs and where they start.
  __device__ __forceinline__ KvSegment sequence(int at, int &length, int &base, int &pairs) const {
    KvSegment g;
    g.b = b0 + at;
    const int first = __builtin_amdgcn_readfirstlane(sm[64 + at]), rows = __builtin_amdgcn_readfirstlane(sm[128 + at]);
    g.seq = kv_sequence(first, first + rows, __builtin_amdgcn_readfirstlane(sm[192 + at]), a.T, a.max_pages, a.page_shift);
    const kv_share h = share_of(g.seq);
    g.steps = h.steps;
    length = __builtin_amdgcn_readfirstlane(kv_length(h, cut));
    pairs = h.blocks * a.H_kv;
    base = __builtin_amdgcn_readfirstlane(sm[at]) - pairs * length;
    return g;
  }
  // The pair at pos, pos < end, and its steps before `end`. Steps past a padded pair's own: none (from >= to).
  __device__ __forceinline__ KvSegment at(int pos, int end) {
    const int l = find(pos);
    if (l < 0) return KvSegment{};
    int length, base, pairs;
    KvSegment g = sequence(l, length, base, pairs);
    const int pair = __builtin_amdgcn_readfirstlane(kv_div(pos - base, length));
    g.start = base + pair * length;
    g.from = pos - g.start;
    g.to = min(g.steps, end - g.start);
    g.rb = __builtin_amdgcn_readfirstlane(kv_div(pair, a.H_kv));
    g.hk = pair - g.rb * a.H_kv;
    if (by_pair()) g.rb = __builtin_amdgcn_readfirstlane(kv_div(pairs, a.H_kv)) - 1 - g.rb;
    return g;
  }
};

}  // namespace mtk
