// 16-bit values into blocks of 32 four-bit values (e2m1) with one power-of-two scale.
//
// The maximum of a block's magnitudes (over the bits: the patterns of a sign-free 16-bit float ascend with its
// value), the smallest power of two that brings it to at most 6, and v_cvt_scalef32_pk's division by it and rounding to
// nearest, ties to the even code: exact but for that one rounding, which is the format's. Magnitudes are first limited to the
// largest value of the grid that the 16-bit type holds, so that nothing reads back as an infinity; a block with a NaN or an
// infinity gets scale 255 and reads as NaN.
#pragma once

#include "grouped.hpp"
#include "kv_device.hpp"

namespace mtk {

// A lane's 8 values of a block that it shares with its three neighbours: their codes, the even place in the low half of a byte,
// and the block's scale byte.
template <int DT>
__device__ __forceinline__ void mx_quantise8(u32x4 v, uint32_t &codes, int &byte) {
  constexpr uint32_t kInf = DT == DT_F16 ? 0x7C00u : 0x7F80u;
  constexpr uint32_t kMost = DT == DT_F16 ? 0x7A00u : 0x7F40u;  // 1.5 times the largest power of two
  // the two halves of a word apart, then together
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  auto two = [](uint32_t x) { return __builtin_bit_cast(u16x2, x); };
  auto most = [&](uint32_t x, uint32_t y) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(two(x), two(y))); };
  constexpr uint32_t kMag = 0x7fff7fffu;
  uint32_t top = most(most(v[0] & kMag, v[1] & kMag), most(v[2] & kMag, v[3] & kMag));
  top = most(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));  // lane ^ 1
  top = most(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));  // lane ^ 2
  top = max(top & 0xffffu, top >> 16);
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
  // the largest magnitude is 1.m * 2^(exponent - 127); 6 = 1.5 * 2^2: a larger mantissa than 1.5's carries into the exponent
  const int e = max((int)((f + 0x3fffffu) >> 23) - 2, 1);
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

}  // namespace mtk
