// Rows of K and V into a paged cache in few bits, and back (kv_cache.h has the layout).
//
// Write: of each block of 32 dims the magnitudes' maximum (over the bits: the patterns of a sign-free 16-bit float
// ascend with its value), the smallest power of two that brings it into the format's range (6 for e2m1, 448 for
// e4m3), and v_cvt_scalef32_pk's division by it and rounding to nearest, ties to even. All of it is exact but the
// one rounding. Magnitudes are first limited to the largest value of the format's grid that the 16-bit type holds,
// so that nothing reads back as an infinity. A block with a NaN or an infinity gets scale 255 and reads as NaN.
// Read: value times scale, two per instruction, exact.
//
// `parts` wavefronts share a row: a lane has 8 dims (16 bytes of K or V) at a time, 4 neighbours a block.
#include "kv_device.hpp"

namespace mtk {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Maximum over the 4 lanes of a block.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));  // lane ^ 1
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));  // lane ^ 2
}

// Where a lane's item (8 dims of K or V of one head of a row) lies.
template <int FMT>
struct KvItem {
  int d, head, blk, quarter, v;
  __device__ __forceinline__ KvItem(const mtk_kv_move_kargs &a, int it) {
    quarter = it & 3;
    int rest = it >> 2;
    blk = rest % a.blocks;
    rest /= a.blocks;
    head = rest % a.H_kv;
    v = rest / a.H_kv;
    d = 32 * blk + 8 * quarter;
  }
  // byte offsets of the codes and the scale in the cache
  __device__ __forceinline__ void place(const mtk_kv_move_kargs &a, int page, int off, uint64_t &code, uint64_t &scale) const {
    const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
    const uint64_t base = ((uint64_t)(uint32_t)page * a.H_kv + head) * kv_region_bytes(FMT, a.blocks, a.page_shift);
    constexpr uint32_t kQ = FMT == KV_FP4 ? 4 : 8;
    code = base + (v ? row_b << a.page_shift : 0u) + off * row_b + blk * 4 * kQ + quarter * kQ;
    scale = base + ((2 * row_b + (v ? a.blocks : 0)) << a.page_shift) + off * a.blocks + blk;
  }
};

// The row of this wavefront, and where it lies in the cache (page -1: nowhere).
__device__ __forceinline__ int kv_place(const mtk_kv_move_kargs &a, int t, int lane, int &off) {
  const int b = seq_of_row(a, t, lane);
  off = 0;
  if (b < 0) return -2;
  const kv_seq s = load_seq(a, b);
  const int64_t pos = s.pos0 + (t - s.first);
  off = (int)(pos & ((1 << a.page_shift) - 1));
  return __builtin_amdgcn_readfirstlane(kv_page(a.table + (size_t)b * a.max_pages, pos, a.n_pages, a.max_pages, a.page_shift));
}

template <int DT, int FMT>
__device__ __forceinline__ void kv_write(const mtk_kv_move_kargs &a) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t64 = w / a.parts;
  if (t64 >= a.T) return;
  const int t = (int)t64, part = (int)(w - t64 * a.parts);
  int off;
  const int page = kv_place(a, t, lane, off);
  if (page < 0) return;
  const int items = 8 * a.H_kv * a.blocks;
  constexpr uint32_t kInf = DT == DT_F16 ? 0x7C00u : 0x7F80u;
  constexpr uint32_t kMost = DT == DT_F16 ? (FMT == KV_FP4 ? 0x7A00u : 0x7B80u) : (FMT == KV_FP4 ? 0x7F40u : 0x7F70u);
  for (int it = part * 64 + lane; it < items; it += 64 * a.parts) {  // items are whole blocks of 4 lanes
    const KvItem<FMT> x(a, it);
    u32x4 v = u32x4{0u, 0u, 0u, 0u};
    const uint16_t *src = (const uint16_t *)(x.v ? a.V : a.K) + (size_t)t * (x.v ? a.ld_v : a.ld_k) + (size_t)x.head * a.D + x.d;
    if (x.d < a.D) v = *(const u32x4 *)src;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = v[i] & 0x7fff7fffu;
      top = max(top, max(m & 0xffffu, m >> 16));
    }
    top = block_max(top);
    const bool bad = top >= kInf;
    if (top > kMost) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = min(v[i] & 0x7fffu, kMost), hi = min((v[i] >> 16) & 0x7fffu, kMost);
        v[i] = bad ? 0u : (v[i] & 0x80008000u) | lo | (hi << 16);
      }
      top = kMost;
    }
    const uint32_t f = __builtin_bit_cast(uint32_t, from_bits<DT>(top));
    // the largest magnitude is 1.m * 2^(exponent - 127); 6 = 1.5 * 2^2, 448 = 1.75 * 2^8
    int byte = FMT == KV_FP4 ? (int)(f >> 23) - 2 + ((f & 0x7fffffu) > 0x400000u) : (int)(f >> 23) - 8 + ((f & 0x7fffffu) > 0x600000u);
    byte = max(byte, 1);
    const float scale = scale_of((uint32_t)byte);
    uint64_t code, at;
    x.place(a, page, off, code, at);
    char *c = (char *)a.cache;
    auto pair = [&](uint32_t w) {
      if constexpr (DT == DT_F16)
        return __builtin_bit_cast(f16x2, w);
      else
        return __builtin_bit_cast(bf16x2, w);
    };
    if constexpr (FMT == KV_FP4) {
      uint32_t r = 0;
      const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
      if constexpr (DT == DT_F16) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, pair(v0), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, pair(v1), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, pair(v2), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, pair(v3), scale, 3);
      } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(v0), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(v1), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(v2), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair(v3), scale, 3);
      }
      *(uint32_t *)(c + code) = r;
    } else {
      s16x2 r0 = s16x2{0, 0}, r1 = s16x2{0, 0};
      const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
      if constexpr (DT == DT_F16) {
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r0, pair(v0), scale, false);
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r0, pair(v1), scale, true);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r1, pair(v2), scale, false);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r1, pair(v3), scale, true);
      } else {
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r0, pair(v0), scale, false);
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r0, pair(v1), scale, true);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r1, pair(v2), scale, false);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r1, pair(v3), scale, true);
      }
      *(u32x2 *)(c + code) = u32x2{__builtin_bit_cast(uint32_t, r0), __builtin_bit_cast(uint32_t, r1)};
    }
    if (x.quarter == 0) *(uint8_t *)(c + at) = (uint8_t)(bad ? kNanScale : byte);
  }
}

template <int DT, int FMT>
__device__ __forceinline__ void kv_read(const mtk_kv_move_kargs &a) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t64 = w / a.parts;
  if (t64 >= a.T) return;
  const int t = (int)t64, part = (int)(w - t64 * a.parts);
  int off;
  const int page = kv_place(a, t, lane, off);
  if (page == -2) return;  // no sequence's row: left as it was
  const int items = 8 * a.H_kv * a.blocks;
  constexpr uint32_t kNan = DT == DT_F16 ? 0x7E007E00u : 0x7FC07FC0u;
  const char *c = (const char *)a.cache;
  for (int it = part * 64 + lane; it < items; it += 64 * a.parts) {
    const KvItem<FMT> x(a, it);
    if (x.d >= a.D) continue;
    u32x4 v = u32x4{kNan, kNan, kNan, kNan};
    if (page >= 0) {
      uint64_t code, at;
      x.place(a, page, off, code, at);
      uint32_t words[kWords8<FMT>];
      if constexpr (FMT == KV_FP4) {
        words[0] = *(const uint32_t *)(c + code);
      } else {
        const u32x2 y = *(const u32x2 *)(c + code);
        words[0] = y.x;
        words[1] = y.y;
      }
      const uint32_t s = *(const uint8_t *)(c + at);
      if (s != kNanScale) v = values8<DT, FMT>(words, scale_of(s));
    }
    uint16_t *dst = (uint16_t *)(x.v ? a.V : a.K) + (size_t)t * (x.v ? a.ld_v : a.ld_k) + (size_t)x.head * a.D + x.d;
    *(u32x4 *)dst = v;
  }
}

}  // namespace mtk

using namespace mtk;

#define MTK_KV_MOVE(FMT, NAME, DT)                                                                     \
  extern "C" __global__ void __launch_bounds__(256) mtk_kv_write_##NAME(const mtk_kv_move_kargs a) {   \
    kv_write<DT, FMT>(a);                                                                              \
  }                                                                                                    \
  extern "C" __global__ void __launch_bounds__(256) mtk_kv_read_##NAME(const mtk_kv_move_kargs a) {    \
    kv_read<DT, FMT>(a);                                                                               \
  }
MTK_KV_MOVE(KV_FP4, fp4_f16, DT_F16)
MTK_KV_MOVE(KV_FP4, fp4_bf16, DT_BF16)
MTK_KV_MOVE(KV_FP8, fp8_f16, DT_F16)
MTK_KV_MOVE(KV_FP8, fp8_bf16, DT_BF16)
