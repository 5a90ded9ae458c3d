// 16-bit rows into blocks of 32 four-bit values with one power-of-two scale each, and back (mx.h has the layout).
//
// Quantise: mx_quantise.hpp has the mathematics. Places past K are zeros, up to a whole number of 256.
// Dequantise: code times scale, two per instruction, exact (f16 values below 2^-14: to the nearest subnormal).
//
// A lane has 8 places of a row (16 bytes in 16 bits, 4 in codes), 4 neighbours a block, 32 a K-tile; a wavefront two K-tiles
// of MX_ROWS rows, whose loads are all in flight at once.
#include "grouped.hpp"
#include "mx.h"
#include "mx_quantise.hpp"

namespace mtk {

constexpr int kMxRows = 4;  // rows of a wavefront

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
  const AnyRows src((const uint16_t *)a.src + p.r0 * a.ld, n, a.ld, a.K);
  u32x4 v[kMxRows];
  uint32_t e[kMxRows] = {};
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) src.load<2>(i, p.k, v[i], e[i]);
  const int lane = threadIdx.x & 63;
  char *codes = (char *)a.codes + p.r0 * mx_row_bytes(a.k_tiles) + (int64_t)p.kt * 128 + 4 * (lane & 31);
  uint32_t bytes = 0;  // of the block's scales, row by row
#pragma unroll
  for (int i = 0; i < kMxRows; ++i) {
    uint32_t c;
    int byte;
    mx_quantise8<DT>(src.take(i, p.k, v[i], e[i]), c, byte);
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
