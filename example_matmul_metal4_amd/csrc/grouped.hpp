// Products grouped by expert: C[t] = A[t] op(B_e) + bias_e for the rows t of group e, and the weights' gradients
// dB_e = sum over its rows of dC[t] x A[t]. Few rows run the GEMM's quarter tiles (quarter.hpp): here a workgroup finds its
// group and tile, and narrows operands and buffer ranges to them. Large tiles are in expert_tiles.hpp.
//
// Where the groups start lies on the device, so a launch's grid is what ascending groups need at most, and workgroups past
// what they do need end at once. Every wavefront looks its tile up by itself: the groups' block counts, 64 groups to a
// window of lanes, summed over the lanes; the tiles of all groups, one group after another, are dealt to the XCDs in
// contiguous runs of the count that there is (not of the grid's), so that neighbours share an L2 and no XCD goes idle.
// Rows behind a group's end are out of the tile's buffer range: they read as zeros, whatever the next group holds.
#pragma once

#include "groups.h"
#include "quarter.hpp"
#include "tile_direct.hpp"

namespace mtk {

// 16 and 8 bytes at any alignment that their elements have: one access, which the hardware splits where it crosses a line.
struct __attribute__((packed, aligned(2))) Chunk {
  u32x4 v;
};
struct __attribute__((packed, aligned(4))) Pair {
  f32x2 v;
};

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int lanes_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// A window of 64 groups in the lanes.
struct GroupWindow {
  group_rows g;
  int end;  // blocks of the window's groups up to this lane's
  __device__ __forceinline__ GroupWindow(const int32_t *row_start, int E, int T, int block, int e0) {
    const int e = e0 + (threadIdx.x & 63);
    g = e < E ? group_of(row_start[e], row_start[e + 1], T) : group_rows{0, 0};
    end = lanes_scan((g.rows + block - 1) / block);
  }
  __device__ __forceinline__ int blocks() const { return __builtin_amdgcn_readlane(end, 63); }
};

// A workgroup's group, and which of the group's blocks x tiles_n tiles it has.
struct GroupTile {
  int e = -1;  // none
  int first, rows, blocks, t;
};

template <int BLOCK>
__device__ __forceinline__ GroupTile group_tile(const int32_t *row_start, int E, int T, int tiles_n) {
  GroupTile r;
  GroupWindow w(row_start, E, T, BLOCK, 0);
  int total = w.blocks();
#pragma unroll 1
  for (int e0 = 64; e0 < E; e0 += 64) total += GroupWindow(row_start, E, T, BLOCK, e0).blocks();
  total *= tiles_n;
  if ((int)blockIdx.x >= total) return r;
  int id = xcd_remap(blockIdx.x, total);
#pragma unroll 1
  for (int e0 = 0;;) {
    const uint64_t in = __ballot(w.end * tiles_n > id);
    if (in) {
      const int i = __builtin_ctzll(in);
      const int end = __builtin_amdgcn_readlane(w.end, i);
      r.e = e0 + i;
      r.first = __builtin_amdgcn_readlane(w.g.first, i);
      r.rows = __builtin_amdgcn_readlane(w.g.rows, i);
      r.blocks = (r.rows + BLOCK - 1) / BLOCK;
      r.t = id - (end - r.blocks) * tiles_n;
      return r;
    }
    id -= w.blocks() * tiles_n;
    e0 += 64;
    if (e0 >= E) return r;  // never: id < total
    w = GroupWindow(row_start, E, T, BLOCK, e0);
  }
}

// Bytes from the dword in which an operand starts to the end of its last element's dword.
__device__ __forceinline__ uint32_t range_of(const void *p, uint32_t exact, bool any) {
  return (exact + (any ? (uint32_t)(uintptr_t)p & 2u : 0u) + 3u) & ~3u;
}

// The part of the GEMM's arguments that a tile of group e takes: `rows` rows of A from `row` on, one block at most.
template <int BLOCK, bool ANY>
__device__ __forceinline__ mtk_tile_args group_args(const mtk_grouped_kargs &g, int e, int row, int rows) {
  mtk_tile_args a{};
  rows = min(rows, BLOCK);
  a.A = (const uint16_t *)g.A + (size_t)row * (size_t)g.lda;
  a.B = (const uint16_t *)g.B + (size_t)e * (size_t)g.b_stride;
  a.bias = (const uint16_t *)g.bias + (size_t)e * (size_t)g.N;
  a.C = (uint16_t *)g.C + (size_t)row * (size_t)g.ldc;
  a.M = rows;
  a.N = g.N;
  a.K = g.K;
  a.lda = g.lda;
  a.ldb = g.ldb;
  a.ldc = g.ldc;
  a.a_bytes = range_of(a.A, ((uint32_t)(rows - 1) * (uint32_t)g.lda + (uint32_t)g.K) * 2u, ANY);
  a.b_bytes = range_of(a.B, g.b_exact, ANY);
  a.k_tiles = a.k_tiles_per_split = g.k_tiles;
  a.split_k = 1;
  a.has_bias = g.has_bias;
  return a;
}

// Row block and column of tile t of a group, groups of 4 row blocks at a time as in the GEMM.
template <int BM, int BN>
__device__ __forceinline__ TileAt tile_at(int t, int blocks, int tiles_n) {
  const int group = kGroupM * tiles_n;
  const int first = (t / group) * kGroupM;
  const int gm = min(blocks - first, kGroupM);
  return TileAt{(first + (t % group) % gm) * BM, (t % group) / gm * BN, false};
}

template <int DT, bool BN, bool ANY, int W>
__device__ __forceinline__ void grouped_quarter(const mtk_grouped_kargs &g) {
  const GroupTile gt = group_tile<64>(g.row_start, g.E, g.T, g.tiles_n);
  if (gt.e < 0) return;
  const TileAt at = tile_at<64, 64>(gt.t, gt.blocks, g.tiles_n);
  const mtk_tile_args a = group_args<64, ANY>(g, gt.e, gt.first + at.m0, gt.rows - at.m0);
  using A = std::conditional_t<ANY, QuarterAny<false>, QuarterOp<false, false>>;
  quarter_tile<DT, A, BN, ANY, W, true>(a, A{}, TileAt{0, at.n0, g.b_once && gt.blocks == 1});
}

// Gradients: K runs over the group's rows, of which both operands hold K rows of M and of N columns. A group without a row has
// zeros.
template <bool ANY>
__device__ __forceinline__ mtk_tile_args grad_args(const mtk_grouped_kargs &g, int e) {
  mtk_tile_args a{};
  const int start = __builtin_amdgcn_readfirstlane(g.row_start[e]), next = __builtin_amdgcn_readfirstlane(g.row_start[e + 1]);
  const group_rows r = group_of(start, next, g.T);
  a.A = (const uint16_t *)g.A + (size_t)r.first * (size_t)g.lda;
  a.B = (const uint16_t *)g.B + (size_t)r.first * (size_t)g.ldb;
  const size_t out = (size_t)e * (size_t)g.M * (size_t)g.N;
  a.C = (uint16_t *)g.C + out;
  a.partial = g.C32 ? g.C32 + out : nullptr;
  a.M = g.M;
  a.N = g.N;
  a.K = r.rows;
  a.lda = g.lda;
  a.ldb = g.ldb;
  a.ldc = g.N;
  a.a_bytes = r.rows ? range_of(a.A, ((uint32_t)(r.rows - 1) * (uint32_t)g.lda + (uint32_t)g.M) * 2u, ANY) : 0u;
  a.b_bytes = r.rows ? range_of(a.B, ((uint32_t)(r.rows - 1) * (uint32_t)g.ldb + (uint32_t)g.N) * 2u, ANY) : 0u;
  a.k_tiles = a.k_tiles_per_split = (r.rows + kBK - 1) / kBK;
  a.split_k = 1;
  return a;
}

template <int DT, bool ANY, int W>
__device__ __forceinline__ void grouped_grad_quarter(const mtk_grouped_kargs &g) {
  // an XCD has 16 neighbours of every 128 tiles: those of a large group are spread over all of them
  const int tiles = g.tiles_m * g.tiles_n;
  const int id = group_nth_tile((int)blockIdx.x & 127, 128, (int)blockIdx.x >> 7, (int)gridDim.x, 0).tile, e = id / tiles;
  const mtk_tile_args a = grad_args<ANY>(g, e);
  using A = std::conditional_t<ANY, QuarterAny<true>, QuarterOp<true, false>>;
  quarter_tile<DT, A, true, ANY, W, true>(a, A{}, tile_at<64, 64>(id - e * tiles, g.tiles_m, g.tiles_n));
}

// dbias_e[n] = sum over the group's rows of dC[t][n]: 64 columns per workgroup, one per lane; its 16 wavefronts take every 16th
// row, 8 of them in flight at a time, and their sums in 32 bits are added in wavefront order. Latency bounds it: 343 rows of the
// largest of 24 groups, 1023 columns: 8 wavefronts with two columns per lane 15.3 us.
constexpr int kBiasWaves = 16, kBiasCols = 64;
template <int DT>
__device__ __forceinline__ void grouped_bias_grad(const mtk_grouped_kargs &g) {
  __shared__ float sums[kBiasWaves][kBiasCols];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e = blockIdx.x / g.tiles_n, n0 = (blockIdx.x - e * g.tiles_n) * kBiasCols;
  const int start = __builtin_amdgcn_readfirstlane(g.row_start[e]), next = __builtin_amdgcn_readfirstlane(g.row_start[e + 1]);
  const group_rows r = group_of(start, next, g.T);
  const uint16_t *at = (const uint16_t *)g.A + (size_t)(r.first + wave) * (size_t)g.lda + min(n0 + lane, g.N - 1);
  const size_t step = (size_t)kBiasWaves * (size_t)g.lda;
  float s = 0.0f;
  int i = wave;
  constexpr int kAhead = 8;
  for (; i + (kAhead - 1) * kBiasWaves < r.rows; i += kAhead * kBiasWaves, at += kAhead * step) {
    uint16_t v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = at[j * step];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) s += from_bits<DT>(v[j]);
  }
  if (i < r.rows) {  // the rest, rows past the last read again and not added
    uint16_t v[kAhead];
    const int n = (r.rows - i + kBiasWaves - 1) / kBiasWaves;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = at[min(j, n - 1) * step];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) s += j < n ? from_bits<DT>(v[j]) : 0.0f;
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && n0 + lane < g.N) {
    float t = sums[0][lane];
#pragma unroll
    for (int w = 1; w < kBiasWaves; ++w) t += sums[w][lane];
    const size_t out = (size_t)e * (size_t)g.N + (size_t)(n0 + lane);
    if (g.C32)
      g.C32[out] = t;
    else
      ((uint16_t *)g.C)[out] = to_bits<DT>(t);
  }
}

}  // namespace mtk
