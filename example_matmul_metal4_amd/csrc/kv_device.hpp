// Device helpers of the kernels on the paged cache in few bits (kv_cache.h): conversions of codes, sums over a
// wavefront, and the search for a workgroup's share of the batch.
#pragma once

#include "device.hpp"
#include "kv_cache.h"

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
__device__ __forceinline__ float wave_sum(float v) {
  auto step = [](float x, auto ctrl, auto mask) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                                     decltype(mask)::value, 0xf, false));
  };
  using std::integral_constant;
  v = step(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  v = step(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  v = step(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// A wavefront's view of the batch: which sequence has unit `id` (or packed row `id`).
struct KvUnit {
  int b = -1;     // sequence, -1: none
  int total = 0;  // units of the launch
  int base = 0;   // the sequence's first unit
  kv_seq seq;
  kv_share share;
};

template <typename A>
__device__ __forceinline__ kv_seq load_seq(const A &a, int b) {
  if (b >= a.B) return kv_sequence(0, 0, 0, 0, a.max_pages, a.page_shift);
  return kv_sequence(a.row_start[b], a.row_start[b + 1], a.kv_len[b], a.T, a.max_pages, a.page_shift);
}

// The sequence that holds packed row t (every lane gets it), or -1.
template <typename A>
__device__ __forceinline__ int seq_of_row(const A &a, int t, int lane) {
  int found = -1;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    const uint64_t in = __ballot(b < a.B && a.row_start[min(b, a.B)] <= t && t < a.row_start[min(b, a.B - 1) + 1]);
    if (in) {
      found = b0 + __builtin_ctzll(in);
      break;
    }
  }
  return __builtin_amdgcn_readfirstlane(found);
}

// The shares of the sequences in kernels of ROWS rows per block and STEP keys per step, and the sequence that
// unit(total) falls into, or sequence `want_b` if that is not negative. One wavefront's lanes hold 64 sequences.
template <int ROWS, int STEP, typename F>
__device__ __forceinline__ KvUnit find_unit(const mtk_kv_attn_kargs &a, int lane, int want_b, F &&unit) {
  const int G = a.G;
  KvUnit u;
  auto share_of = [&](const kv_seq &s) { return kv_blocks(s, a.S_q, G, ROWS, STEP, a.rows_above, a.rows_most); };
  // work -> steps per workgroup
  float work = 0.0f;
  kv_seq s0 = load_seq(a, lane);
  kv_share h0 = share_of(s0);
  work = (float)h0.blocks * (float)h0.steps;
  for (int b0 = 64; b0 < a.B; b0 += 64) {
    const kv_share h = share_of(load_seq(a, b0 + lane));
    work += (float)h.blocks * (float)h.steps;
  }
  const float each = ceilf(wave_sum(work) * (float)a.H_kv / (float)a.units);
  int c = max(a.least, each < 1e9f ? (int)each : 1000000000);
  if (a.B <= 64) {
    int scan = 0;
#pragma unroll 1
    for (int i = 0;; ++i) {
      kv_split(&h0, c);
      scan = wave_scan(h0.blocks * h0.splits * a.H_kv);
      u.total = __builtin_amdgcn_readlane(scan, 63);
      if (u.total <= a.units || i == 2) break;
      c = kv_next_c(c, u.total, a.units);
    }
    const int id = unit(u.total);
    const uint64_t past = want_b >= 0 ? 1ull << want_b : __ballot(scan > id);
    if (!past || (want_b < 0 && id < 0)) return u;
    const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
    u.b = at;
    u.base = __builtin_amdgcn_readlane(scan - h0.blocks * h0.splits * a.H_kv, at);
  } else {
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      kv_share h = share_of(load_seq(a, b0 + lane));
      kv_split(&h, c);
      u.total += __builtin_amdgcn_readlane(wave_scan(h.blocks * h.splits * a.H_kv), 63);
    }
    const int id = unit(u.total);
    if (want_b < 0 && (id < 0 || id >= u.total)) return u;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      kv_share h = share_of(load_seq(a, b0 + lane));
      kv_split(&h, c);
      const int n = h.blocks * h.splits * a.H_kv, scan = before + wave_scan(n);
      const uint64_t past = want_b >= 0 ? (want_b - b0 < 64 ? 1ull << (want_b - b0) : 0ull) : __ballot(scan > id);
      if (past) {
        const int at = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
        u.b = b0 + at;
        u.base = __builtin_amdgcn_readlane(scan - n, at);
        break;
      }
      before = __builtin_amdgcn_readlane(scan, 63);
    }
    if (u.b < 0) return u;
  }
  u.seq = load_seq(a, u.b);
  u.share = share_of(u.seq);
  kv_split(&u.share, c);
  return u;
}

}  // namespace mtk
