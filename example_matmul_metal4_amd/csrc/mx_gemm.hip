// Products of rows in few bits: C = A B_e^T + bias_e, A and B in blocks of 32 e2m1 values with one power-of-two scale (mx.h),
// fp32 accumulate on the scaled MFMA, which multiplies the codes' values exactly.
#include "expert_tiles.hpp"
#include "mx_quantise.hpp"

namespace mtk {

// The tile of this workgroup: rows of A, and the group. One group of all rows where there is no row_start.
template <int BLOCK>
__device__ __forceinline__ GroupTile mx_tile(const mtk_mx_gemm_kargs &g) {
  if (g.row_start) return group_tile<BLOCK>(g.row_start, g.E, g.T, g.tiles_n);
  GroupTile r;
  r.e = 0;
  r.first = 0;
  r.rows = g.T;
  r.blocks = (g.T + BLOCK - 1) / BLOCK;
  r.t = xcd_remap(blockIdx.x, gridDim.x);
  return r;
}

// 32 MB rows x 64 columns, the K-tiles over the workgroup's 8 wavefronts as in quarter.hpp: each has its own part of LDS, no
// barrier until their sums are added, in wavefront order. QUANT: A are 16-bit rows, which every workgroup brings into the format
// for itself as it stages them, a few instructions per row that the loads of B cover where rows are few (the plan has both sides).
template <int DT, int MB, bool QUANT>
__device__ __forceinline__ void mx_few(const mtk_mx_gemm_kargs &g) {
  constexpr int W = 8, ROWS = 32 * MB, kScaleB = QUANT ? ROWS * 8 : 0, kWaveB = (ROWS + 64) * 128 + kScaleB;
  static_assert(!QUANT || MB == 1, "registers of the rows in flight");
  static_assert(MB * 8192 <= kWaveB, "the sums fit the staging area");
  __shared__ __attribute__((aligned(1024))) char smem[W * kWaveB];
  const GroupTile gt = mx_tile<ROWS>(g);
  if (gt.e < 0) return;
  const TileAt at = tile_at<ROWS, 64>(gt.t, gt.blocks, g.tiles_n);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = min(gt.rows - at.m0, ROWS), cols = min(g.N - at.n0, 64);
  const bool b_once = !QUANT && g.b_once && gt.blocks == 1;
  const int64_t first = gt.first + at.m0;
  const MxOperand A(QUANT ? nullptr : g.A, QUANT ? nullptr : g.a_scales, first, QUANT ? 0 : rows, g.T, g.k_tiles);
  const MxOperand B(g.B, g.b_scales, (int64_t)gt.e * g.N + at.n0, cols, (int64_t)g.E * g.N, g.k_tiles);

  char *la = smem + wave * kWaveB, *lb = la + ROWS * 128, *ls = lb + 8192;
  const uint32_t lane_a = (uint32_t)(lane >> 3) * A.row_b + 16u * (uint32_t)(lane & 7);
  const uint32_t lane_b = (uint32_t)(lane >> 3) * B.row_b + 16u * (uint32_t)(lane & 7);
  const uint32_t lane_s = 8u * (uint32_t)(lane & 31) + 4u * (uint32_t)(lane >> 5);
  // QUANT: load i has rows 2 i and 2 i + 1, 8 places per lane
  const int half = lane >> 5, place = 8 * (lane & 31), pairs = (rows + 1) >> 1;
  const AnyRows src(QUANT ? (const uint16_t *)g.A + first * g.lda : nullptr, rows, g.lda, g.K);
  u32x4 va[QUANT ? 16 : 4 * MB] = {}, vb[8];
  uint32_t ve[16] = {};
  uint32_t na[MB], nb[2];
  const int turn = g.turns.on ? group_turn(group_turn_place(gt.e, at.n0 / 64, g.turns), g.k_tiles) : 0;
  auto load = [&](int k) {
    const int kt = group_turned(k, turn, g.k_tiles);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t off = lane_b + (uint32_t)i * 8u * B.row_b + (uint32_t)kt * 128u;
      vb[i] = b_once ? __builtin_amdgcn_raw_buffer_load_b128(B.codes, off, 0, 2) : buf_load16(B.codes, off);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) nb[i] = buf_load4(B.scales, lane_s + 256u * (uint32_t)i + (uint32_t)kt * B.tile_s);
    if constexpr (QUANT) {
      static_for<0, 16>([&](auto i) {  // (rows that are not there are out of range)
        if (i < pairs) src.load(2 * i + half, kt * 256 + place, va[i], ve[i]);
      });
    } else {
#pragma unroll
      for (int i = 0; i < 4 * MB; ++i) va[i] = buf_load16(A.codes, lane_a + (uint32_t)i * 8u * A.row_b + (uint32_t)kt * 128u);
#pragma unroll
      for (int i = 0; i < MB; ++i) na[i] = buf_load4(A.scales, lane_s + 256u * (uint32_t)i + (uint32_t)kt * A.tile_s);
    }
  };
  f32x16 acc[MB][2] = {};
  int kt = wave;
  if (kt < g.k_tiles) load(kt);
  for (; kt < g.k_tiles; kt += W) {
    uint32_t sa[MB], sb[2];
    if constexpr (QUANT) {
      const int k = group_turned(kt, turn, g.k_tiles) * 256 + place;
      static_for<0, 16>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        if (i < pairs) {
          uint32_t code;
          int byte;
          mx_quantise8<DT>(src.take(2 * i + half, k, va[i], ve[i]), code, byte);
          const int row = 2 * i + half, block = place >> 5;
          *(uint32_t *)(la + lds_off(row, block) + 4 * (lane & 3)) = code;
          if ((lane & 3) == 0) *(uint8_t *)(ls + 8 * row + block) = (uint8_t)byte;
        }
      });
    } else {
#pragma unroll
      for (int i = 0; i < 4 * MB; ++i) *(u32x4 *)(la + lds_off(8 * i + (lane >> 3), lane & 7)) = va[i];
#pragma unroll
      for (int i = 0; i < MB; ++i) sa[i] = na[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *(u32x4 *)(lb + lds_off(8 * i + (lane >> 3), lane & 7)) = vb[i];
#pragma unroll
    for (int i = 0; i < 2; ++i) sb[i] = nb[i];
    if (kt + W < g.k_tiles) load(kt + W);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (QUANT) sa[0] = *(const uint32_t *)(ls + lane_s);
    static_for<0, 4>([&](auto s_c) {
      constexpr int s = decltype(s_c)::value;
      u32x4 fa[MB], fb[2];
#pragma unroll
      for (int i = 0; i < MB; ++i) fa[i] = *(const u32x4 *)(la + lds_off(32 * i + (lane & 31), 4 * (lane >> 5) + s));
#pragma unroll
      for (int i = 0; i < 2; ++i) fb[i] = *(const u32x4 *)(lb + lds_off(32 * i + (lane & 31), 4 * (lane >> 5) + s));
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_mx32<s>(fa[i], fb[j], acc[i][j], sa[i], sb[j]);
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // ---- add the wavefronts' sums, in wavefront order: accumulator quads parked as [block][quad][lane], 16 bytes each
  f32x4 *park = (f32x4 *)(smem + wave * kWaveB);  // own region
#pragma unroll
  for (int b = 0; b < 2 * MB; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16 &x = acc[b >> 1][b & 1];
      park[(4 * b + q) * 64 + lane] = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    }
  __syncthreads();
  const uint16_t *bias = (const uint16_t *)g.bias + (size_t)gt.e * (size_t)g.N;
  uint16_t *C = (uint16_t *)g.C + (size_t)first * (size_t)g.ldc + at.n0;
#pragma unroll
  for (int it = tid; it < 512 * MB; it += 64 * W) {
    const int b = it >> 8, q = (it >> 6) & 3, l = it & 63;
    const int row = 32 * (b >> 1) + 8 * q + 4 * (l >> 5), col = 32 * (b & 1) + (l & 31);
    if (col >= cols || row >= rows) continue;
    f32x4 s = *(const f32x4 *)(smem + it * 16);
#pragma unroll
    for (int w = 1; w < W; ++w) s += *(const f32x4 *)(smem + w * kWaveB + it * 16);
    const float bv = g.has_bias ? from_bits<DT>(bias[at.n0 + col]) : 0.0f;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (row + r < rows) C[(size_t)(row + r) * (size_t)g.ldc + col] = to_bits<DT>(v[r] + bv);
  }
}

}  // namespace mtk

using namespace mtk;

#define MTK_MX_GEMM(NAME, DT)                                                                                    \
  extern "C" __global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))                   \
  mtk_mx_gemm_##NAME##_64(const mtk_mx_gemm_kargs g) {                                                           \
    mx_few<DT, 2, false>(g);                                                                                     \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))                   \
  mtk_mx_gemm_##NAME##_32(const mtk_mx_gemm_kargs g) {                                                           \
    mx_few<DT, 1, false>(g);                                                                                     \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))                   \
  mtk_mx_gemm_##NAME##_32q(const mtk_mx_gemm_kargs g) {                                                          \
    mx_few<DT, 1, true>(g);                                                                                      \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(512) mtk_mx_gemm_##NAME##_256(const mtk_mx_gemm_kargs g) {        \
    expert_tiles<Mx<DT>, 256, 256, 2, 4, TileRows<256, 8, true>, TileRows<256, 8, true>>(MxTiles<256, 256>(g));  \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) mtk_mx_gemm_##NAME##_128(const mtk_mx_gemm_kargs g) {        \
    expert_tiles<Mx<DT>, 128, 128, 2, 2, TileRows<128, 4, true>, TileRows<128, 4, true>>(MxTiles<128, 128>(g));  \
  }
MTK_MX_GEMM(f16, DT_F16)
MTK_MX_GEMM(bf16, DT_BF16)
