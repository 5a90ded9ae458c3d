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

// Some 16-bit rows of K places, ld apart, as they lie in memory: at any 2-byte alignment. What lies behind the last row's end is out of
// the buffer's range.
struct AnyRows {
  rsrc_t buf;
  uint32_t mis, step;  // bytes from the buffer's start to the first row, and between rows
  int K;
  bool odd;            // rows start in the middle of dwords
  __device__ __forceinline__ AnyRows(const void *first, int rows, int64_t ld, int K_) : K(K_) {
    const uint32_t bytes = ((uint32_t)(rows - 1) * (uint32_t)ld + (uint32_t)K_) * 2u;
    buf = make_rsrc_any(first, range_of(first, bytes, true), mis);
    step = (uint32_t)ld * 2u;
    odd = mis != 0 || (ld & 1) != 0;
  }
  __device__ __forceinline__ uint32_t at(int row, int k) const { return (uint32_t)row * step + (uint32_t)k * 2u + mis; }
  // The 8 places of a row from k on, in two steps, so that many loads are in flight: the dwords that hold them ...
  // (POLICY 2: past the caches)
  template <int POLICY = 0>
  __device__ __forceinline__ void load(int row, int k, u32x4 &v, uint32_t &e) const {
    const uint32_t off = k < K ? at(row, k) : kOOBAny;
    v = __builtin_amdgcn_raw_buffer_load_b128(buf, off & ~3u, 0, POLICY);
    if (odd) e = buf_load4(buf, (off & ~3u) + 16u);
  }
  // ... and the places themselves, zeros from K on.
  __device__ __forceinline__ u32x4 take(int row, int k, u32x4 v, uint32_t e) const {
    if (odd) {
      const uint32_t sh = (at(row, k) & 2u) << 3;
      v = u32x4{__builtin_amdgcn_alignbit(v.y, v.x, sh), __builtin_amdgcn_alignbit(v.z, v.y, sh), __builtin_amdgcn_alignbit(v.w, v.z, sh),
                __builtin_amdgcn_alignbit(e, v.w, sh)};
    }
    return K - k < 8 ? keep_halves(v, K - k) : v;
  }
};

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
  return TileAt{(first + (t % group) % gm) * BM, (t % group) / gm * BN, false, 0};
}

template <int DT, bool BN, bool ANY, int W>
__device__ __forceinline__ void grouped_quarter(const mtk_grouped_kargs &g) {
  const GroupTile gt = group_tile<64>(g.row_start, g.E, g.T, g.tiles_n);
  if (gt.e < 0) return;
  const TileAt at = tile_at<64, 64>(gt.t, gt.blocks, g.tiles_n);
  const mtk_tile_args a = group_args<64, ANY>(g, gt.e, gt.first + at.m0, gt.rows - at.m0);
  using A = std::conditional_t<ANY, QuarterAny<false>, QuarterOp<false, false>>;
  quarter_tile<DT, A, BN, ANY, W, true>(a, A{}, TileAt{0, at.n0, g.b_once && gt.blocks == 1, g.turns.on ? group_turn(group_turn_place(gt.e, at.n0 / 64, g.turns), g.K / kBK) : 0});
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

// dbias_e[n] = sum over the group's rows of dC[t][n]: 64 columns from n0 on per workgroup, 8 neighbours a lane, 64 rows a step of a
// wavefront, all in flight at once, the steps over the W wavefronts. Sums in 32 bits: a lane's rows in order, then rows apart by 1, 2
// and 4 of 8, then the wavefronts in order. Latency bounds it where groups have few rows, HBM where a launch of its own reads dC
// again.
template <int DT, int W>
__device__ __forceinline__ void bias_columns(const mtk_grouped_kargs &g, const void *dC, int ld, int N, void *out, int e, int n0) {
  __shared__ float sums[W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int start = __builtin_amdgcn_readfirstlane(g.row_start[e]), next = __builtin_amdgcn_readfirstlane(g.row_start[e + 1]);
  const group_rows r = group_of(start, next, g.T);
  const int c = lane & 7, r0 = lane >> 3, k = n0 + 8 * c;
  const AnyRows src((const uint16_t *)dC + (size_t)r.first * (size_t)ld, max(r.rows, 1), ld, N);
  float s[8] = {};
  for (int i = 64 * wave; i < r.rows; i += 64 * W) {
    u32x4 v[8];
    uint32_t x[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = i + 8 * j + r0;
      src.load(row, row < r.rows ? k : N, v[j], x[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32x4 w = src.take(i + 8 * j + r0, k, v[j], x[j]);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        s[2 * h] += from_bits<DT>((uint16_t)(w[h] & 0xffffu));
        s[2 * h + 1] += from_bits<DT>((uint16_t)(w[h] >> 16));
      }
    }
  }
  float t = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float y = s[j];
    y += __shfl_xor(y, 8);
    y += __shfl_xor(y, 16);
    y += __shfl_xor(y, 32);
    t = r0 == j ? y : t;  // column 8 c + r0
  }
  if constexpr (W > 1) {
    sums[wave][lane] = t;
    __syncthreads();
    if (wave > 0) return;
    t = sums[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) t += sums[w][lane];
  }
  const int col = n0 + 8 * c + r0;
  if (col >= N) return;
  const size_t at = (size_t)e * (size_t)N + (size_t)col;
  if (g.C32)
    ((float *)out)[at] = t;
  else
    ((uint16_t *)out)[at] = to_bits<DT>(t);
}

// The bias's gradient as a launch of its own, beside large tiles. 4, 8 and 16 wavefronts, us of the launch: 8192 rows over 16 groups of 4096
// columns 16.0, 15.6, 17.8; 16384 over 2 of 1024 40.7, 24.1, 24.7; 1000 over 24 of 1024 6.9, 6.5, 7.7; 30000 of one of 4096 -, 114, 118.
constexpr int kBiasWaves = 8;
template <int DT>
__device__ __forceinline__ void grouped_bias_grad(const mtk_grouped_kargs &g) {
  const int e = blockIdx.x / g.tiles_n;
  bias_columns<DT, kBiasWaves>(g, g.A, g.lda, g.N, g.C32 ? (void *)g.C32 : g.C, e, 64 * (blockIdx.x - e * g.tiles_n));
}

// The first g.lead workgroups (a multiple of 8, or none) have the bias's gradient: dC is A (has_bias 1) or B (2).
template <int DT, bool ANY, int W>
__device__ __forceinline__ void grouped_grad_quarter(const mtk_grouped_kargs &g) {
  int block = blockIdx.x;
  if (block < g.lead) {
    const bool a = g.has_bias == 1;
    const int N = a ? g.M : g.N, across = (N + 63) >> 6, e = block / across;
    if (e < g.E) bias_columns<DT, W>(g, a ? g.A : g.B, a ? g.lda : g.ldb, N, const_cast<void *>(g.bias), e, 64 * (block - e * across));
    return;
  }
  block -= g.lead;
  // an XCD has 16 neighbours of every 128 tiles: those of a large group are spread over all of them
  const int tiles = g.tiles_m * g.tiles_n;
  const int id = group_nth_tile(block & 127, 128, block >> 7, (int)gridDim.x - g.lead, 0).tile, e = id / tiles;
  const mtk_tile_args a = grad_args<ANY>(g, e);
  using A = std::conditional_t<ANY, QuarterAny<true>, QuarterOp<true, false>>;
  quarter_tile<DT, A, true, ANY, W, true>(a, A{}, tile_at<64, 64>(id - e * tiles, g.tiles_m, g.tiles_n));
}

}  // namespace mtk
