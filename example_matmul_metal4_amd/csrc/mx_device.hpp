// Device helpers of the products of rows in few bits (mx.h): the scaled MFMA, and a group's operands.
#pragma once

#include "grouped.hpp"
#include "mx.h"

namespace mtk {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 32x32x64, fp32 accumulate: a lane has one block of 32 codes of row lane % 32 of either operand (16 bytes), and byte SEL of
// its scale word is that block's. Lanes 0 to 31 and 32 to 63 have two blocks of K, which ones is free as long as A and B agree.
template <int SEL>
__device__ __forceinline__ f32x16 mfma_mx32(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}

// ds_read_b32 as inline asm, for code with direct-to-LDS loads in flight (device.hpp): the caller waits for it.
template <int OFF>
__device__ __forceinline__ uint32_t ds_read_b32_at(uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  uint32_t w;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(w) : "v"(addr), "i"(OFF));
  return w;
}

// Buffers of `rows` rows of an operand, the first of them row `row` of `all`: codes, and scales with offsets
// kt * all * 8 + r * 8 from that row.
struct MxOperand {
  rsrc_t codes, scales;
  uint32_t row_b;   // bytes of a row's codes
  uint32_t tile_s;  // bytes of scales from one K-tile to the next
  __device__ __forceinline__ MxOperand(const void *c, const void *s, int64_t row, int rows, int64_t all, int k_tiles) {
    row_b = (uint32_t)mx_row_bytes(k_tiles);
    tile_s = (uint32_t)(all * 8);
    codes = make_rsrc((const char *)c + row * (int64_t)row_b, (uint32_t)rows * row_b);
    // the last K-tile's scales of the last row are the last that is read
    scales = make_rsrc((const char *)s + row * 8, (uint32_t)(k_tiles - 1) * tile_s + (uint32_t)rows * 8);
  }
};

}  // namespace mtk
