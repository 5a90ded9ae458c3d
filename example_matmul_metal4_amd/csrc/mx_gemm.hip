// Products of rows in few bits: C = A B_e^T + bias_e, A and B in blocks of 32 e2m1 values with one power-of-two scale (mx.h),
// fp32 accumulate on the scaled MFMA, which multiplies the codes' values exactly.
#include "expert_tiles.hpp"

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

// 64x64 tiles, the K-tiles over the workgroup's 8 wavefronts as in quarter.hpp.
template <int DT>
__device__ __forceinline__ void mx_quarter(const mtk_mx_gemm_kargs &g) {
  constexpr int W = 8, kWaveB = 16384;
  __shared__ __attribute__((aligned(1024))) char smem[W * kWaveB];
  const GroupTile gt = mx_tile<64>(g);
  if (gt.e < 0) return;
  const TileAt at = tile_at<64, 64>(gt.t, gt.blocks, g.tiles_n);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = min(gt.rows - at.m0, 64), cols = min(g.N - at.n0, 64);
  const MxOperand A(g.A, g.a_scales, gt.first + at.m0, rows, g.T, g.k_tiles);
  const MxOperand B(g.B, g.b_scales, (int64_t)gt.e * g.N + at.n0, cols, (int64_t)g.E * g.N, g.k_tiles);

  char *la = smem + wave * kWaveB, *lb = la + 8192;
  const uint32_t lane_a = (uint32_t)(lane >> 3) * A.row_b + 16u * (uint32_t)(lane & 7);
  const uint32_t lane_b = (uint32_t)(lane >> 3) * B.row_b + 16u * (uint32_t)(lane & 7);
  const uint32_t lane_s = 8u * (uint32_t)(lane & 31) + 4u * (uint32_t)(lane >> 5);
  u32x4 va[8], vb[8];
  uint32_t sa[2], sb[2], na[2], nb[2];
  auto load = [&](int kt) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      va[i] = buf_load16(A.codes, lane_a + (uint32_t)i * 8u * A.row_b + (uint32_t)kt * 128u);
      vb[i] = buf_load16(B.codes, lane_b + (uint32_t)i * 8u * B.row_b + (uint32_t)kt * 128u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      na[i] = buf_load4(A.scales, lane_s + 256u * (uint32_t)i + (uint32_t)kt * A.tile_s);
      nb[i] = buf_load4(B.scales, lane_s + 256u * (uint32_t)i + (uint32_t)kt * B.tile_s);
    }
  };
  f32x16 acc[2][2] = {};
  int kt = wave;
  if (kt < g.k_tiles) load(kt);
  for (; kt < g.k_tiles; kt += W) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      *(u32x4 *)(la + lds_off(8 * i + (lane >> 3), lane & 7)) = va[i];
      *(u32x4 *)(lb + lds_off(8 * i + (lane >> 3), lane & 7)) = vb[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sa[i] = na[i];
      sb[i] = nb[i];
    }
    if (kt + W < g.k_tiles) load(kt + W);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    static_for<0, 4>([&](auto s_c) {
      constexpr int s = decltype(s_c)::value;
      u32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *(const u32x4 *)(la + lds_off(32 * i + (lane & 31), 4 * (lane >> 5) + s));
        fb[i] = *(const u32x4 *)(lb + lds_off(32 * i + (lane & 31), 4 * (lane >> 5) + s));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_mx32<s>(fa[i], fb[j], acc[i][j], sa[i], sb[j]);
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // ---- add the wavefronts' sums, in wavefront order: accumulator quads parked as [block][quad][lane], 16 bytes each
  f32x4 *park = (f32x4 *)(smem + wave * kWaveB);  // own region
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16 &x = acc[b >> 1][b & 1];
      park[(4 * b + q) * 64 + lane] = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    }
  __syncthreads();
  const uint16_t *bias = (const uint16_t *)g.bias + (size_t)gt.e * (size_t)g.N;
  uint16_t *C = (uint16_t *)g.C + (size_t)(gt.first + at.m0) * (size_t)g.ldc + at.n0;
#pragma unroll
  for (int it = tid; it < 1024; it += 64 * W) {
    f32x4 s = *(const f32x4 *)(smem + it * 16);
#pragma unroll
    for (int w = 1; w < W; ++w) s += *(const f32x4 *)(smem + w * kWaveB + it * 16);
    const int b = it >> 8, q = (it >> 6) & 3, l = it & 63;
    const int row = 32 * (b >> 1) + 8 * q + 4 * (l >> 5), col = 32 * (b & 1) + (l & 31);
    if (col >= cols) continue;
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
    mx_quarter<DT>(g);                                                                                           \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(512) mtk_mx_gemm_##NAME##_256(const mtk_mx_gemm_kargs g) {        \
    expert_tiles<Mx<DT>, 256, 256, 2, 4, TileRows<256, 8, true>, TileRows<256, 8, true>>(MxTiles<256, 256>(g));  \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) mtk_mx_gemm_##NAME##_128(const mtk_mx_gemm_kargs g) {        \
    expert_tiles<Mx<DT>, 128, 128, 2, 2, TileRows<128, 4, true>, TileRows<128, 4, true>>(MxTiles<128, 128>(g));  \
  }
MTK_MX_GEMM(f16, DT_F16)
MTK_MX_GEMM(bf16, DT_BF16)
