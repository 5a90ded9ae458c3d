// 16-bit rows into blocks of 32 four-bit values with one power-of-two scale each, and back (mx.h has the layout).
//
// Quantise: the maximum of a block's magnitudes (over the bits: the patterns of a sign-free 16-bit float ascend with its
// value), the smallest power of two that brings it to at most 6, and v_cvt_scalef32_pk's division by it and rounding to
// nearest, ties to the even code: exact but for that one rounding, which is the format's. Magnitudes are first limited to the
// largest value of the grid that the 16-bit type holds, so that nothing reads back as an infinity; a block with a NaN or an
// infinity gets scale 255 and reads as NaN. Places past K are zeros, up to a whole number of 256.
// Dequantise: code times scale, two per instruction, exact (f16 values below 2^-14: to the nearest subnormal).
//
// A lane has 8 places of a row (16 bytes in 16 bits, 4 in codes), 4 neighbours a block, 32 a K-tile; a wavefront two K-tiles
// of MX_ROWS rows, whose loads are all in flight at once.
#include "grouped.hpp"
#include "kv_device.hpp"
#include "mx.h"

namespace mtk {

constexpr int kMxRows = 4;  // rows of a wavefront

template <int DT>
__device__ __forceinline__ void mx_quantise8(u32x4 v, uint32_t &codes, int &byte) {
  constexpr uint32_t kInf = DT == DT_F16 ? 0x7C00u : 0x7F80u;
  constexpr uint32_t kMost = DT == DT_F16 ? 0x7A00u : 0x7F40u;  // 1.5 times the largest power of two
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = v[i] & 0x7fff7fffu;
    top = max(top, max(m & 0xffffu, m >> 16));
  }
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));  // lane ^ 2
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
  // the largest magnitude is 1.m * 2^(exponent - 127); 6 = 1.5 * 2^2
  const int e = max((int)(f >> 23) - 2 + ((f & 0x7fffffu) > 0x400000u), 1);
  const float scale = scale_of((uint32_t)e);
  const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
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
  codes = r;
  byte = bad ? kNanScale : e;
}

// A wavefront's two K-tiles (pair `kp` of the row) of rows r0 .. r0 + kMxRows - 1, lane by lane: 8 places from k on.
struct MxPlace {
  int64_t r0;
  int k, kt, block;  // K-tile, and block in it
  __device__ __forceinline__ explicit MxPlace(const mtk_mx_rows_kargs &a) {
    const int pairs = (a.k_tiles + 1) >> 1;
    const int64_t w = (int64_t)xcd_remap(blockIdx.x, gridDim.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t group = w / pairs;
    const int kp = (int)(w - group * pairs);
    const int lane = threadIdx.x & 63;
    r0 = group * kMxRows;
    kt = 2 * kp + (lane >> 5);
    k = kt * 256 + 8 * (lane & 31);
    block = (lane & 31) >> 2;
  }
};

template <int DT>
__device__ __forceinline__ void mx_quantise(const mtk_mx_rows_kargs &a) {
  const MxPlace p(a);
  if (p.r0 >= a.R) return;
  const int n = (int)min((int64_t)kMxRows, a.R - p.r0);
  const uint16_t *src = (const uint16_t *)a.src + p.r0 * a.ld + p.k;
  u32x4 v[kMxRows];
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) v[i] = u32x4{0u, 0u, 0u, 0u};
  if (p.k + 8 <= a.K) {
#pragma unroll
    for (int i = 0; i < kMxRows; ++i)
      if (i < n) v[i] = ((const Chunk *)(src + (int64_t)i * a.ld))->v;
  } else if (p.k < a.K) {
#pragma unroll
    for (int i = 0; i < kMxRows; ++i) {
      if (i >= n) break;
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = p.k + j < a.K ? src[(int64_t)i * a.ld + j] : 0u;
      v[i] = u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
    }
  }
  const int lane = threadIdx.x & 63;
  char *codes = (char *)a.codes + p.r0 * mx_row_bytes(a.k_tiles) + (int64_t)p.kt * 128 + 4 * (lane & 31);
  uint32_t bytes = 0;  // of the block's scales, row by row
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) {
    uint32_t c;
    int byte;
    mx_quantise8<DT>(v[i], c, byte);
    bytes |= (uint32_t)byte << (8 * i);
    if (i < n && p.kt < a.k_tiles) *(uint32_t *)(codes + i * mx_row_bytes(a.k_tiles)) = c;
  }
  // A K-tile's scales of the four rows are 32 bytes in a row: lane 8 * row + block of each half stores one, all in one instruction.
  static_assert(kMxRows == 4, "32 bytes for 32 lanes");
  bytes = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * ((lane & 32) + 4 * (lane & 7)), (int)bytes);
  const int row = (lane >> 3) & 3;
  if (row < n && p.kt < a.k_tiles)
    ((uint8_t *)a.scales)[((int64_t)p.kt * a.R + p.r0 + row) * 8 + (lane & 7)] = (uint8_t)(bytes >> (8 * row));
}

template <int DT>
__device__ __forceinline__ void mx_dequantise(const mtk_mx_rows_kargs &a) {
  const MxPlace p(a);
  if (p.r0 >= a.R || p.k >= a.K) return;
  const int n = (int)min((int64_t)kMxRows, a.R - p.r0);
  const char *codes = (const char *)a.codes + p.r0 * mx_row_bytes(a.k_tiles) + (int64_t)p.kt * 128 + 4 * (threadIdx.x & 31);
  const uint8_t *scales = (const uint8_t *)a.scales + ((int64_t)p.kt * a.R + p.r0) * 8 + p.block;
  uint32_t c[kMxRows], s[kMxRows];
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) {
    c[i] = s[i] = 0;
    if (i < n) {
      c[i] = *(const uint32_t *)(codes + i * mx_row_bytes(a.k_tiles));
      s[i] = scales[8 * i];
    }
  }
  constexpr uint32_t kNan = DT == DT_F16 ? 0x7E007E00u : 0x7FC07FC0u;
  uint16_t *dst = (uint16_t *)a.dst + p.r0 * a.ld + p.k;
  const bool whole = p.k + 8 <= a.K;
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) {
    if (i >= n) break;
    u32x4 v = u32x4{kNan, kNan, kNan, kNan};
    if (s[i] != kNanScale) v = values8<DT, KV_FP4>(&c[i], scale_of(s[i]));
    uint16_t *at = dst + (int64_t)i * a.ld;
    if (whole) {
      ((Chunk *)at)->v = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = v[j >> 1];
        if (p.k + j < a.K) at[j] = (uint16_t)(j & 1 ? w >> 16 : w);
      }
    }
  }
}

}  // namespace mtk

using namespace mtk;

#define MTK_MX_ROWS(NAME, DT)                                                                                \
  extern "C" __global__ void __launch_bounds__(256) mtk_mx_quantize_##NAME(const mtk_mx_rows_kargs a) {      \
    mx_quantise<DT>(a);                                                                                      \
  }                                                                                                          \
  extern "C" __global__ void __launch_bounds__(256) mtk_mx_dequantize_##NAME(const mtk_mx_rows_kargs a) {    \
    mx_dequantise<DT>(a);                                                                                    \
  }
MTK_MX_ROWS(f16, DT_F16)
MTK_MX_ROWS(bf16, DT_BF16)
