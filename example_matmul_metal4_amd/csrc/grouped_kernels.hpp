// The kernels of products grouped by expert for one element type. A translation unit defines
//   MTK_GROUPED_DT        DT_F16 or DT_BF16
//   MTK_GROUPED_NAME(x)   the kernel name for suffix x
// and includes this file once.
//   nt_*, nn_*   C = A op(B_e) with B_e [N][K] / [K][N]; *_256, *_128: square tiles of the GEMM's pipeline, *_64: quarter
//   grad_*       the weights' gradients, likewise; bias_grad: the bias's
//   *_any        rows at any 2-byte alignment (odd leading dimensions)
#pragma once

#include "expert_tiles.hpp"

namespace mtk_grouped_ops {
using namespace mtk;
using El = Half<MTK_GROUPED_DT>;
// 256x256 tiles: 8 wavefronts (2 x 4, 128 x 64 each, two per SIMD); 128x128: 4 (2 x 2), two workgroups per CU
__device__ __forceinline__ void nt_256(const mtk_grouped_kargs &g) {
  expert_tiles<El, 256, 256, 2, 4, TileRows<256, 8>, TileRows<256, 8>>(ForwardTiles<256, 256, false>(g));
}
__device__ __forceinline__ void nn_256(const mtk_grouped_kargs &g) {
  expert_tiles<El, 256, 256, 2, 4, TileRows<256, 8>, TileCols<256, 8>>(ForwardTiles<256, 256, true>(g));
}
__device__ __forceinline__ void nt_128(const mtk_grouped_kargs &g) {
  expert_tiles<El, 128, 128, 2, 2, TileRows<128, 4>, TileRows<128, 4>>(ForwardTiles<128, 128, false>(g));
}
__device__ __forceinline__ void nn_128(const mtk_grouped_kargs &g) {
  expert_tiles<El, 128, 128, 2, 2, TileRows<128, 4>, TileCols<128, 4>>(ForwardTiles<128, 128, true>(g));
}
__device__ __forceinline__ void grad_256(const mtk_grouped_kargs &g) {
  expert_tiles<El, 256, 256, 2, 4, TileCols<256, 8>, TileCols<256, 8>>(GradTiles<256, 256>(g));
}
__device__ __forceinline__ void grad_128(const mtk_grouped_kargs &g) {
  expert_tiles<El, 128, 128, 2, 2, TileCols<128, 4>, TileCols<128, 4>>(GradTiles<128, 128>(g));
}
}  // namespace mtk_grouped_ops

#define MTK_GROUPED(NAME, THREADS, ...)                                                                     \
  extern "C" __global__ void __launch_bounds__(THREADS) MTK_GROUPED_NAME(NAME)(const mtk_grouped_kargs g) { \
    __VA_ARGS__(g);                                                                                          \
  }
// quarter tiles, K-tiles over W wavefronts: 8, or 4 in two workgroups per CU, or 1 in eight
#define MTK_GROUPED_QUARTER(NAME, W, ...)                                                           \
  extern "C" __global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2)))   \
  MTK_GROUPED_NAME(NAME##_w##W)(const mtk_grouped_kargs g) {                                        \
    mtk::__VA_ARGS__, W>(g);                                                                         \
  }
#define MTK_GROUPED_QUARTERS(W)                                                      \
  MTK_GROUPED_QUARTER(nt_64, W, grouped_quarter<MTK_GROUPED_DT, false, false)         \
  MTK_GROUPED_QUARTER(nn_64, W, grouped_quarter<MTK_GROUPED_DT, true, false)          \
  MTK_GROUPED_QUARTER(nt_64_any, W, grouped_quarter<MTK_GROUPED_DT, false, true)      \
  MTK_GROUPED_QUARTER(nn_64_any, W, grouped_quarter<MTK_GROUPED_DT, true, true)       \
  MTK_GROUPED_QUARTER(grad_64, W, grouped_grad_quarter<MTK_GROUPED_DT, false)         \
  MTK_GROUPED_QUARTER(grad_64_any, W, grouped_grad_quarter<MTK_GROUPED_DT, true)
MTK_GROUPED_QUARTERS(8)
MTK_GROUPED_QUARTERS(4)
MTK_GROUPED_QUARTERS(1)

MTK_GROUPED(nt_256, 512, mtk_grouped_ops::nt_256)
MTK_GROUPED(nn_256, 512, mtk_grouped_ops::nn_256)
MTK_GROUPED(nt_128, 256, mtk_grouped_ops::nt_128)
MTK_GROUPED(nn_128, 256, mtk_grouped_ops::nn_128)
MTK_GROUPED(grad_256, 512, mtk_grouped_ops::grad_256)
MTK_GROUPED(grad_128, 256, mtk_grouped_ops::grad_128)
MTK_GROUPED(bias_grad, 512, mtk::grouped_bias_grad<MTK_GROUPED_DT>)
