// The kernels of products grouped by expert for one element type. A translation unit defines
//   MTK_GROUPED_DT        DT_F16 or DT_BF16
//   MTK_GROUPED_NAME(x)   the kernel name for suffix x
// and includes this file once.
//   nt_*, nn_*   C = A op(B_e) with B_e [N][K] / [K][N]; *_256, *_128: square tiles of the GEMM's pipeline, *_64: quarter
//   grad_*       the weights' gradients, likewise; bias_grad: the bias's
//   *_any        rows at any 2-byte alignment (odd leading dimensions)
#pragma once

#include "grouped.hpp"

namespace mtk_grouped_ops {
using R256 = mtk::OpRows<256, 8>;
using C256 = mtk::OpColsT<256, 8>;
using R128 = mtk::OpRows<128, 4>;
using C128 = mtk::OpColsT<128, 4>;
}  // namespace mtk_grouped_ops

#define MTK_GROUPED(NAME, THREADS, ...)                                                                     \
  extern "C" __global__ void __launch_bounds__(THREADS) MTK_GROUPED_NAME(NAME)(const mtk_grouped_kargs g) { \
    mtk::__VA_ARGS__(g);                                                                                     \
  }
// quarter tiles: one workgroup of 8 wavefronts per CU, whose registers they may all have
#define MTK_GROUPED_QUARTER(NAME, ...)                                                              \
  extern "C" __global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))      \
  MTK_GROUPED_NAME(NAME)(const mtk_grouped_kargs g) {                                               \
    mtk::__VA_ARGS__(g);                                                                             \
  }

MTK_GROUPED(nt_256, 512, grouped_direct<MTK_GROUPED_DT, 256, 2, 4, mtk_grouped_ops::R256, mtk_grouped_ops::R256>)
MTK_GROUPED(nn_256, 512, grouped_direct<MTK_GROUPED_DT, 256, 2, 4, mtk_grouped_ops::R256, mtk_grouped_ops::C256>)
MTK_GROUPED(nt_128, 256, grouped_direct<MTK_GROUPED_DT, 128, 2, 2, mtk_grouped_ops::R128, mtk_grouped_ops::R128>)
MTK_GROUPED(nn_128, 256, grouped_direct<MTK_GROUPED_DT, 128, 2, 2, mtk_grouped_ops::R128, mtk_grouped_ops::C128>)
MTK_GROUPED_QUARTER(nt_64, grouped_quarter<MTK_GROUPED_DT, false, false, 8>)
MTK_GROUPED_QUARTER(nn_64, grouped_quarter<MTK_GROUPED_DT, true, false, 8>)
MTK_GROUPED_QUARTER(nt_64_any, grouped_quarter<MTK_GROUPED_DT, false, true, 8>)
MTK_GROUPED_QUARTER(nn_64_any, grouped_quarter<MTK_GROUPED_DT, true, true, 8>)
MTK_GROUPED(grad_256, 512, grouped_grad_direct<MTK_GROUPED_DT, 256, 2, 4, mtk_grouped_ops::C256, mtk_grouped_ops::C256>)
MTK_GROUPED(grad_128, 256, grouped_grad_direct<MTK_GROUPED_DT, 128, 2, 2, mtk_grouped_ops::C128, mtk_grouped_ops::C128>)
MTK_GROUPED_QUARTER(grad_64, grouped_grad_quarter<MTK_GROUPED_DT, false, 8>)
MTK_GROUPED_QUARTER(grad_64_any, grouped_grad_quarter<MTK_GROUPED_DT, true, 8>)
MTK_GROUPED(bias_grad, 512, grouped_bias_grad<MTK_GROUPED_DT>)
