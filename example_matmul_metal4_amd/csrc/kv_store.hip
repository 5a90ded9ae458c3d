// Rows of K and V into a paged cache in few bits, and back (kv_cache.h has the layout).
//
// Write: of each block of 32 dims the magnitudes' maximum (over the bits: the patterns of a sign-free 16-bit float
// ascend with its value), the smallest power of two that brings it into the format's range (6 for e2m1, 448 for
// e4m3), and v_cvt_scalef32_pk's division by it and rounding to nearest, ties to even. All of it is exact but the
// one rounding. Magnitudes are first limited to the largest value of the format's grid that the 16-bit type holds,
// so that nothing reads back as an infinity. A block with a NaN or an infinity gets scale 255 and reads as NaN.
// Read: value times scale, two per instruction, exact.
//
// A lane has 8 dims (16 bytes of K or V), 4 neighbours a block, of up to 4 rows, whose loads are in flight at once; a
// wavefront looks its rows up once (row_start and kv_len of 64 sequences at a time, then the table).
//
// Bound by HBM, few rows by three dependent loads (3.1 us). 32000 rows of 8 heads x 128 dims read back from fp4, by rows
// per wavefront: 1: 67 us, 2: 48, 4: 37.8 (4.4 TB/s), 8: 42, 16: 44; by rows with several of a row's items in flight instead:
// 47.6. Workgroups in XCD order, so that neighbours' partial lines meet in one L2: fp8, 5700 rows x 32 heads x 80 dims,
// written and read back 51.3 -> 48.8 us.
// K and V are loaded past the caches, as nothing reads them again once they are in the cache: that write 30.4 -> 23.8 us,
// with what made the rows before it 92 -> 82 us for 32000 rows. What is read back is stored through the caches: past them
// the kernel takes 27.6 us instead of 37.8, but with its reader 88.3 instead of 86.1 (6000 rows: 22.1 and 18.7).
#include "kv_device.hpp"

namespace mtk {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Maximum over the 4 lanes of a block.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));  // lane ^ 1
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));  // lane ^ 2
}

// n / d, d's multiplier ceil(2^32 / d) (0: d is 1); exact for n * d < 2^32.
__device__ __forceinline__ int div_by(int n, uint32_t mul) { return mul ? (int)__umulhi((uint32_t)n, mul) : n; }

// Where a lane's item (8 dims of K or V of one head of a row) lies in a row of K or V and in a page of the cache.
template <int FMT>
struct KvItem {
  int d, head, quarter, v;
  uint64_t code, scale;  // byte offsets of position 0's codes and scale from the page
  __device__ __forceinline__ KvItem(const mtk_kv_move_kargs &a, int it) {
    const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
    quarter = it & 3;
    const int block = it >> 2, both = div_by(block, a.mul_blocks), blk = block - both * a.blocks;
    v = both >= a.H_kv ? 1 : 0;
    head = both - v * a.H_kv;
    d = 32 * blk + 8 * quarter;
    const uint64_t at = (uint64_t)(uint32_t)head * kv_region_bytes(FMT, a.blocks, a.page_shift);
    constexpr uint32_t kQ = FMT == KV_FP4 ? 4 : 8;
    code = at + (v ? row_b << a.page_shift : 0u) + blk * 4 * kQ + quarter * kQ;
    scale = at + ((2 * row_b + (v ? a.blocks : 0)) << a.page_shift) + blk;
  }
};

// The rows of this wavefront: [t0, t0 + n), items [64 * part, 64 * part + 64) of each; lane i has the page of row t0 + i
// (-1: no page, -2: a row of no sequence) and its place in it.
struct KvRows {
  int t0, n = 0, part, page = -2, off = 0;
  __device__ __forceinline__ KvRows(const mtk_kv_move_kargs &a, int lane) {
    const int64_t w = (int64_t)xcd_remap(blockIdx.x, gridDim.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = w / a.parts;
    part = (int)(w - group * a.parts);
    if (group * a.rows_per_wave >= a.T) return;
    t0 = (int)(group * a.rows_per_wave);
    n = min(a.rows_per_wave, a.T - t0);
    bool open = lane < n;  // this lane's row has no sequence yet
    for (int b0 = 0; b0 < a.B && __ballot(open); b0 += 64) {
      const int b = min(b0 + lane, a.B - 1);
      const kv_seq s = load_seq(a, b);
      const int end = s.first + s.rows;
      uint64_t meets = __ballot(b0 + lane < a.B && s.first < t0 + n && end > t0);
      for (; meets; meets &= meets - 1) {
        const int i = __builtin_ctzll(meets);
        const int first = __builtin_amdgcn_readlane(s.first, i), last = __builtin_amdgcn_readlane(end, i);
        const int len = __builtin_amdgcn_readlane(s.len, i);
        const int t = t0 + lane;
        if (open && t >= first && t < last) {
          const int64_t pos = (int64_t)len - (last - t);
          off = (int)(pos & ((1 << a.page_shift) - 1));
          page = kv_page(a.table + (size_t)(b0 + i) * a.max_pages, pos, a.n_pages, a.max_pages, a.page_shift);
          open = false;
        }
      }
    }
  }
};

// The pages and places of a wavefront's rows, as every lane has them: taken from the lanes that looked them up while all lanes
// run, as lanes without an item leave the code below.
struct KvPlaces {
  int page[KV_MOVE_ROWS], off[KV_MOVE_ROWS];
  __device__ __forceinline__ explicit KvPlaces(const KvRows &rows) {
#pragma unroll
    for (int k = 0; k < KV_MOVE_ROWS; ++k) {
      page[k] = __builtin_amdgcn_readlane(rows.page, k);
      off[k] = __builtin_amdgcn_readlane(rows.off, k);
    }
  }
};

template <int DT, int FMT>
__device__ __forceinline__ void kv_write(const mtk_kv_move_kargs &a) {
  const int lane = threadIdx.x & 63;
  const KvRows rows(a, lane);
  const KvPlaces of(rows);
  const int items = 8 * a.H_kv * a.blocks;
  const uint64_t page_b = kv_region_bytes(FMT, a.blocks, a.page_shift) * (uint64_t)a.H_kv;
  const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
  constexpr uint32_t kInf = DT == DT_F16 ? 0x7C00u : 0x7F80u;
  constexpr uint32_t kMost = DT == DT_F16 ? (FMT == KV_FP4 ? 0x7A00u : 0x7B80u) : (FMT == KV_FP4 ? 0x7F40u : 0x7F70u);
  auto one = [&](const KvItem<FMT> &x, char *at, int off, u32x4 v) {
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
    const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
    char *code = at + x.code + (uint32_t)off * row_b;
    if constexpr (FMT == KV_FP4) {
      uint32_t r = 0;
      if constexpr (DT == DT_F16) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, v0), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, v1), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, v2), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, v3), scale, 3);
      } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, v0), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, v1), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, v2), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, v3), scale, 3);
      }
      *(uint32_t *)code = r;
    } else {
      s16x2 r0 = s16x2{0, 0}, r1 = s16x2{0, 0};
      if constexpr (DT == DT_F16) {
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r0, __builtin_bit_cast(f16x2, v0), scale, false);
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r0, __builtin_bit_cast(f16x2, v1), scale, true);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r1, __builtin_bit_cast(f16x2, v2), scale, false);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r1, __builtin_bit_cast(f16x2, v3), scale, true);
      } else {
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r0, __builtin_bit_cast(bf16x2, v0), scale, false);
        r0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r0, __builtin_bit_cast(bf16x2, v1), scale, true);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r1, __builtin_bit_cast(bf16x2, v2), scale, false);
        r1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r1, __builtin_bit_cast(bf16x2, v3), scale, true);
      }
      *(u32x2 *)code = u32x2{__builtin_bit_cast(uint32_t, r0), __builtin_bit_cast(uint32_t, r1)};
    }
    if (x.quarter == 0) *(uint8_t *)(at + x.scale + (uint32_t)off * (uint32_t)a.blocks) = (uint8_t)(bad ? kNanScale : byte);
  };
  const int it = rows.part * 64 + lane;
  if (it < items) {  // 4 lanes are a whole block
    const KvItem<FMT> x(a, it);
    const bool in = x.d < a.D;
    const uint16_t *src = (const uint16_t *)(x.v ? a.V : a.K) + (size_t)x.head * a.D + x.d;
    const int64_t ld = x.v ? a.ld_v : a.ld_k;
    u32x4 v[KV_MOVE_ROWS];
#pragma unroll
    for (int k = 0; k < KV_MOVE_ROWS; ++k) {
      v[k] = u32x4{0u, 0u, 0u, 0u};
      if (in && k < rows.n) v[k] = __builtin_nontemporal_load((const u32x4 *)(src + (size_t)(rows.t0 + k) * ld));
    }
#pragma unroll
    for (int k = 0; k < KV_MOVE_ROWS; ++k)
      if (k < rows.n && of.page[k] >= 0) one(x, (char *)a.cache + (uint64_t)(uint32_t)of.page[k] * page_b, of.off[k], v[k]);
  }
}

template <int DT, int FMT>
__device__ __forceinline__ void kv_read(const mtk_kv_move_kargs &a) {
  const int lane = threadIdx.x & 63;
  const KvRows rows(a, lane);
  const KvPlaces of(rows);
  const int items = 8 * a.H_kv * a.blocks;
  const uint64_t page_b = kv_region_bytes(FMT, a.blocks, a.page_shift) * (uint64_t)a.H_kv;
  const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
  constexpr uint32_t kNan = DT == DT_F16 ? 0x7E007E00u : 0x7FC07FC0u;
  const int it = rows.part * 64 + lane;
  const KvItem<FMT> x(a, it);
  if (it < items && x.d < a.D) {
    uint16_t *dst = (uint16_t *)(x.v ? a.V : a.K) + (size_t)x.head * a.D + x.d;
    const int64_t ld = x.v ? a.ld_v : a.ld_k;
    uint32_t words[KV_MOVE_ROWS][kWords8<FMT>], s[KV_MOVE_ROWS];
#pragma unroll
    for (int k = 0; k < KV_MOVE_ROWS; ++k) {
      s[k] = kNanScale;
      if (k < rows.n && of.page[k] >= 0) {
        const char *at = (const char *)a.cache + (uint64_t)(uint32_t)of.page[k] * page_b;
        const char *code = at + x.code + (uint32_t)of.off[k] * row_b;
        if constexpr (FMT == KV_FP4) {
          words[k][0] = *(const uint32_t *)code;
        } else {
          const u32x2 y = *(const u32x2 *)code;
          words[k][0] = y.x;
          words[k][1] = y.y;
        }
        s[k] = *(const uint8_t *)(at + x.scale + (uint32_t)of.off[k] * (uint32_t)a.blocks);
      }
    }
#pragma unroll
    for (int k = 0; k < KV_MOVE_ROWS; ++k) {
      if (k >= rows.n || of.page[k] == -2) continue;  // no sequence's row: left as it was
      u32x4 v = u32x4{kNan, kNan, kNan, kNan};
      if (s[k] != kNanScale) v = values8<DT, FMT>(words[k], scale_of(s[k]));
      *(u32x4 *)(dst + (size_t)(rows.t0 + k) * ld) = v;
    }
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
