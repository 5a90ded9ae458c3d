// Layout of rows held in blocks of 32 four-bit values (e2m1) with one power-of-two scale each: plain functions that the host
// runtime and the kernels share.
//
// A row of K values is padded with zeros to k_tiles = ceil(K / 256) tiles of 256. Codes [R][k_tiles][128 bytes], two a byte,
// the even place in the low half: a tile of a row is one 128-byte line. Scales [k_tiles][R][8 bytes]: those of a tile's 8
// blocks, rows of one tile together, so that a product's tile of rows has its scales of a K-tile in one run of bytes. A scale
// byte s stands for 2^(s - 127); 255: the block is NaN.
#ifndef MTK_MX_H
#define MTK_MX_H

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

#define MTK_MX_FN static __host__ __device__ __forceinline__
#else
#define MTK_MX_FN static inline
#endif

MTK_MX_FN int mx_k_tiles(int K) { return K / 256 + (K % 256 != 0); }
MTK_MX_FN int64_t mx_row_bytes(int k_tiles) { return (int64_t)k_tiles * 128; }
MTK_MX_FN uint64_t mx_code_bytes(int64_t R, int k_tiles) { return (uint64_t)R * (uint64_t)mx_row_bytes(k_tiles); }
MTK_MX_FN uint64_t mx_scale_bytes(int64_t R, int k_tiles) { return (uint64_t)R * (uint64_t)k_tiles * 8; }

#endif
