// Output tiles of products grouped by expert, 16-bit or in few bits, as one pipeline that runs from a workgroup's first tile to
// its last: a persistent grid, and no K-tile's loads wait for a tile's end.
//
// A K-tile is 128 bytes of a row (64 places in 16 bits, 256 in 4), or 64 rows of a K-major operand. Two LDS stages, filled by
// direct-to-LDS loads whose lanes are handed the addresses that belong at their bytes, so that swizzles are applied on the
// global side. Four k-steps a K-tile, fragments one k-step ahead in two buffers, all of a step's reads in its first two groups of
// MFMAs. The barrier stands before the last k-step: by then every wavefront has read the stage, and the other one's K-tile has
// landed, whose first fragments are read during that step, while the loads of the K-tile after it go into the free stage. At
// a tile's end these are the next tile's. So an output tile costs its epilogue and nothing else: each wavefront parks 16 rows
// at a time of its part in LDS of its own behind the stages, reads them back along rows and stores 16 bytes per lane, without
// a barrier.
//
// Operands start at the tile's first row (or column), with the range that the tile has of them: what lies behind reads as
// zeros, and the lanes' offsets are the same for all tiles. Every tile has two K-tiles at least, the missing ones zeros (the
// gradients of a group without a row are such a tile).
//
// Row blocks of 32 that a tile does not have are not multiplied, in halves of a wavefront's rows: the two wavefronts of a SIMD
// have the upper and the lower half of the tile, so that a group's last tile takes about the time of its rows.
#pragma once

#include "grouped.hpp"
#include "mx_device.hpp"

namespace mtk {

// ---------------------------------------------------------------- operands

// ROWS rows of 128 bytes per K-tile, staged by NW wavefronts as [ROWS][128]. MX: the 16-byte chunk of lane l at k-step ks is
// 4 * (l / 32) + ks, so that the bytes of its scale word are those of its four steps in order; else 2 * ks + l / 32.
template <int ROWS, int NW, bool MX = false>
struct TileRows {
  static constexpr int kLoads = ROWS / (8 * NW), kBytes = ROWS * 128;
  static constexpr bool kMasked = !MX;  // a partial last K-tile holds the next rows' bytes
  uint32_t off[kLoads];
  __device__ __forceinline__ TileRows(int wave, int lane, uint32_t ld_bytes) {
    const uint32_t cbase = (uint32_t)((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int b = wave * kLoads + q;
      off[q] = (uint32_t)(8 * b + (lane >> 3)) * ld_bytes + 16u * (cbase ^ (uint32_t)(b & 7));
    }
  }
  // K-tile k of an operand that spans `bytes` from its first row
  static __device__ __forceinline__ rsrc_t at(const char *p, uint32_t bytes, int, int, int k, bool there) {
    return make_rsrc(p + (size_t)k * 128, there ? bytes - (uint32_t)k * 128u : 0u);
  }
  // the fragment of k-step KS of 32-row block `blk`
  template <int KS>
  static __device__ __forceinline__ u32x4 frag(uint32_t lds, int blk, int lane) {
    const int t = (lane & 7) ^ ((lane >> 3) & 3) ^ ((MX ? 4 : 1) * (lane >> 5));
    const int c = (MX ? KS : 2 * KS) ^ (4 * (blk & 1));
    return ds_read_b128_at<0>(lds + (uint32_t)(blk * 4096 + (lane & 31) * 128 + ((t ^ c) << 4)));
  }
};

// 64 rows of K of COLS columns per K-tile, as [64][COLS], chunk c of row k at c ^ 4 * (k % 4); read with transposed reads.
template <int COLS, int NW>
struct TileCols {
  static constexpr int kLoads = COLS / (8 * NW), kBytes = COLS * 128;
  static constexpr bool kMasked = false;  // rows past K are out of range: zeros
  static constexpr int kRowB = COLS * 2;
  uint32_t off[kLoads];
  __device__ __forceinline__ TileCols(int wave, int lane, uint32_t ld_bytes) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int byte = (wave * kLoads + q) * 1024 + lane * 16, row = byte / kRowB, pc = (byte % kRowB) / 16;
      off[q] = (uint32_t)row * ld_bytes + 16u * (uint32_t)(pc ^ (4 * (row & 3)));
    }
  }
  // bytes: of a row from the tile's first column on
  static __device__ __forceinline__ rsrc_t at(const char *p, uint32_t bytes, int ld, int K, int k, bool there) {
    const int rows = min(K - 64 * k, 64);
    return make_rsrc(p + (size_t)k * ((size_t)ld * 128), there ? ((uint32_t)(rows - 1) * (uint32_t)ld * 2u + bytes + 3u) & ~3u : 0u);
  }
  template <int KS>
  static __device__ __forceinline__ u32x4 frag(uint32_t lds, int blk, int lane) {
    const int s = lane & 15, h = lane >> 4;
    const int row = 8 * (h >> 1) + (s >> 2), c = (4 * blk + 2 * (h & 1) + ((s & 3) >> 1)) ^ (4 * (s >> 2));
    const uint32_t p = lds + (uint32_t)(row * kRowB + 16 * c + 8 * (s & 1));
    const u32x2 x = ds_read_tr16_at<16 * KS * kRowB>(p), y = ds_read_tr16_at<(16 * KS + 4) * kRowB>(p);
    return u32x4{x.x, x.y, y.x, y.y};
  }
};

// The elements of a product: 16 bits, or four with scales.
template <int DT_>
struct Half {
  static constexpr int DT = DT_;
  static constexpr bool kScales = false;
  template <int KS>
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, uint32_t, uint32_t) {
    return mfma32x32x16<DT>(a, b, c);
  }
};
template <int DT_>
struct Mx {
  static constexpr int DT = DT_;
  static constexpr bool kScales = true;
  template <int KS>
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
    return mfma_mx32<KS>(a, b, c, sa, sb);
  }
};

// ---------------------------------------------------------------- a workgroup's tiles

// Tiles of 256 rows are halved in the last round, as their wavefronts of the lower half share the SIMDs with those of the upper one;
// of 128, each SIMD has one wavefront of a tile, and half of them would have nothing to do.
template <int BM>
__device__ __forceinline__ group_place nth_tile(int i, int total) {
  return group_nth_tile((int)blockIdx.x, (int)gridDim.x, i, total, BM == 256);
}
// What a tile of BM rows of which `left` are left starts at and has, by halves.
template <int BM>
__device__ __forceinline__ int half_first(int half) { return half == 2 ? BM / 2 : 0; }
template <int BM>
__device__ __forceinline__ int half_rows(int half, int left) { return min(left, half ? BM / 2 : BM); }

struct ExpertTile {
  const char *a, *b;         // its first row (column) of the operands
  const char *sa, *sb;       // ... of their scales
  uint32_t a_bytes, b_bytes; // TileRows: from there to the operand's end; TileCols: to the row's end
  int rows, cols;
  char *c;                   // its first output
  const uint16_t *bias;      // of its first column, or null
  int e, first, m, n;        // gradients: its group, the group's first row, and its block of rows and of columns
  int K, k_tiles;            // ... and the group's rows
  int turn;                  // its whole K-tiles are taken from this one on
  bool there;
};

// The groups' row blocks, found from row_start (grouped.hpp); the first 64 groups stay in the lanes.
template <int BM>
struct GroupSearch {
  const int32_t *row_start;
  int E, T, tiles_n, total;
  GroupWindow w;
  __device__ __forceinline__ GroupSearch(const int32_t *rs, int E_, int T_, int tiles_n_)
      : row_start(rs), E(E_), T(T_), tiles_n(tiles_n_), w(rs, E_, T_, BM, 0) {
    total = w.blocks();
#pragma unroll 1
    for (int e0 = 64; e0 < E; e0 += 64) total += GroupWindow(row_start, E, T, BM, e0).blocks();
    total = min(total, (int)group_max_blocks(E, T, BM)) * tiles_n;  // groups that do not ascend cost no more than those that do
  }
  __device__ __forceinline__ GroupTile get(int i, int &half) const {
    GroupTile r;
    const group_place place = nth_tile<BM>(i, total);
    int id = place.tile;
    half = place.half;
    if (id < 0) return r;
    GroupWindow v = w;
#pragma unroll 1
    for (int e0 = 0;;) {
      const uint64_t in = __ballot(v.end * tiles_n > id);
      if (in) {
        const int l = __builtin_ctzll(in);
        r.e = e0 + l;
        r.first = __builtin_amdgcn_readlane(v.g.first, l);
        r.rows = __builtin_amdgcn_readlane(v.g.rows, l);
        r.blocks = (r.rows + BM - 1) / BM;
        r.t = id - (__builtin_amdgcn_readlane(v.end, l) - r.blocks) * tiles_n;
        return r;
      }
      id -= v.blocks() * tiles_n;
      e0 += 64;
      if (e0 >= E) return r;  // never: id < total
      v = GroupWindow(row_start, E, T, BM, e0);
    }
  }
};

// C = A op(B_e) + bias_e
template <int BM, int BN, bool KMAJOR>
struct ForwardTiles {
  static constexpr bool kTurned = !KMAJOR;  // tiles may start at different K-tiles (grouped_plans.hpp: kTurnedRows)
  __device__ __forceinline__ int whole() const { return g.K >> 6; }
  __device__ __forceinline__ int K(const ExpertTile &) const { return g.K; }
  __device__ __forceinline__ int k_tiles(const ExpertTile &) const { return g.k_tiles; }
  static constexpr bool kWarm = false;
  const mtk_grouped_kargs &g;
  GroupSearch<BM> search;
  __device__ __forceinline__ explicit ForwardTiles(const mtk_grouped_kargs &g_) : g(g_), search(g_.row_start, g_.E, g_.T, g_.tiles_n) {}
  __device__ __forceinline__ int lda() const { return g.lda; }
  __device__ __forceinline__ int ldb() const { return g.ldb; }
  __device__ __forceinline__ int ldc() const { return g.ldc; }
  __device__ __forceinline__ bool f32() const { return false; }
  // Through the caches, where the next operator finds them: a product in 4 bits of 4096 x 14336 x 4096 and the launch that reads its
  // outputs 151 us, past them 154.
  __device__ __forceinline__ bool streamed() const { return false; }
  __device__ __forceinline__ ExpertTile get(int i) const {
    ExpertTile t{};
    int half;
    const GroupTile gt = search.get(i, half);
    if (gt.e < 0) return t;
    const TileAt at = tile_at<BM, BN>(gt.t, gt.blocks, g.tiles_n);
    const int m0 = at.m0 + half_first<BM>(half), row = gt.first + m0;
    t.rows = half_rows<BM>(half, gt.rows - m0);
    t.there = t.rows > 0;
    if (!t.there) return t;
    t.cols = min(g.N - at.n0, BN);
    t.a = (const char *)g.A + (size_t)row * ((size_t)g.lda * 2);
    t.a_bytes = (((uint32_t)(t.rows - 1) * (uint32_t)g.lda + (uint32_t)g.K) * 2u + 3u) & ~3u;
    t.b = (const char *)g.B + (size_t)gt.e * ((size_t)g.b_stride * 2);
    if constexpr (KMAJOR) {
      t.b += (size_t)at.n0 * 2;
      t.b_bytes = (uint32_t)(g.N - at.n0) * 2u;
    } else {
      t.b += (size_t)at.n0 * ((size_t)g.ldb * 2);
      t.b_bytes = (((uint32_t)(t.cols - 1) * (uint32_t)g.ldb + (uint32_t)g.K) * 2u + 3u) & ~3u;
    }
    t.c = (char *)g.C + ((size_t)row * (size_t)g.ldc + (size_t)at.n0) * 2;
    t.bias = g.has_bias ? (const uint16_t *)g.bias + (size_t)gt.e * (size_t)g.N + at.n0 : nullptr;
    if constexpr (kTurned) t.turn = g.turns.on ? group_turn(group_turn_place(gt.e, at.n0 / BN, g.turns), whole()) : 0;
    return t;
  }
};

// Gradients of the weights: K runs over the group's rows, of which both operands hold K rows of M and of N columns.
//
// A round's workgroups have one group or few, with few K-tiles each, and write as much as they read: the first K-tiles of a new group
// would come from HBM behind the last round's outputs. So the workgroups ask for the group's rows while they are busy with the one
// before it (warm), two K-tiles before its end, each for its part of the columns that its tile has: rows i * tiles_n + n of A's,
// i * tiles_m + m of B's, a lane for a line of 128 bytes. 8192 rows over 16 groups of 4096 x 4096: inputs in HBM 340 -> 306 us, in the
// last-level cache 293 -> 294. (Forward products that ask for later K-tiles of their weights are slower: 306 -> 330.)
template <int BM, int BN>
struct GradTiles {
  static constexpr bool kTurned = false;
  static constexpr bool kWarm = BM == 256;
  const mtk_grouped_kargs &g;
  __device__ __forceinline__ explicit GradTiles(const mtk_grouped_kargs &g_) : g(g_) {}
  __device__ __forceinline__ int K(const ExpertTile &t) const { return t.K; }
  __device__ __forceinline__ int k_tiles(const ExpertTile &t) const { return t.k_tiles; }
  __device__ __forceinline__ int lda() const { return g.lda; }
  __device__ __forceinline__ int ldb() const { return g.ldb; }
  __device__ __forceinline__ int ldc() const { return g.N; }
  __device__ __forceinline__ bool f32() const { return g.C32 != nullptr; }
  __device__ __forceinline__ bool streamed() const { return true; }  // gradients: nothing reads them soon
  __device__ __forceinline__ ExpertTile get(int i) const {
    ExpertTile t{};
    const int tiles = g.tiles_m * g.tiles_n;
    const group_place place = nth_tile<BM>(i, g.E * tiles);
    if (place.tile < 0) return t;
    const int e = place.tile / tiles;
    TileAt at = tile_at<BM, BN>(place.tile - e * tiles, g.tiles_m, g.tiles_n);
    at.m0 += half_first<BM>(place.half);
    t.rows = half_rows<BM>(place.half, g.M - at.m0);
    t.there = t.rows > 0;
    if (!t.there) return t;
    const int start = __builtin_amdgcn_readfirstlane(g.row_start[e]), next = __builtin_amdgcn_readfirstlane(g.row_start[e + 1]);
    const group_rows r = group_of(start, next, g.T);
    t.cols = min(g.N - at.n0, BN);
    t.K = r.rows;
    t.k_tiles = (r.rows + 63) / 64;
    t.a = (const char *)g.A + ((size_t)r.first * (size_t)g.lda + (size_t)at.m0) * 2;
    t.a_bytes = (uint32_t)(g.M - at.m0) * 2u;
    t.b = (const char *)g.B + ((size_t)r.first * (size_t)g.ldb + (size_t)at.n0) * 2;
    t.b_bytes = (uint32_t)(g.N - at.n0) * 2u;
    const size_t out = (size_t)e * (size_t)g.M * (size_t)g.N + (size_t)at.m0 * (size_t)g.N + (size_t)at.n0;
    t.c = g.C32 ? (char *)g.C32 + out * 4 : (char *)g.C + out * 2;
    t.e = e;
    t.first = r.first;
    t.m = at.m0 / BM;
    t.n = at.n0 / BN;
    return t;
  }
  // Where a wavefront asks (4 of them in A, 4 in B), and its lanes' offsets for tile t.
  __device__ __forceinline__ rsrc_t warm(int wave) const {
    const uint32_t ld = (uint32_t)(wave < 4 ? g.lda : g.ldb), width = (uint32_t)(wave < 4 ? g.M : g.N);
    return make_rsrc(wave < 4 ? g.A : g.B, (((uint32_t)(g.T - 1) * ld + width) * 2u) & ~3u);
  }
  __device__ __forceinline__ uint32_t warm_off(const ExpertTile &t, int wave, int lane) const {
    const bool a = wave < 4;
    const int i = 16 * (wave & 3) + (lane >> 2), row = a ? i * g.tiles_n + t.n : i * g.tiles_m + t.m, col = 64 * (lane & 3);
    if (row >= t.K || col >= (a ? t.rows : t.cols)) return kOOBAny;
    return ((uint32_t)(t.first + row) * (uint32_t)(a ? g.lda : g.ldb) + (uint32_t)((a ? t.m * BM : t.n * BN) + col)) * 2u;
  }
};

// C = A B_e^T + bias_e, both in few bits; one group of all rows where there is no row_start.
template <int BM, int BN>
struct MxTiles {
  static constexpr bool kTurned = true;
  __device__ __forceinline__ int whole() const { return g.k_tiles; }
  __device__ __forceinline__ int K(const ExpertTile &) const { return g.K; }
  __device__ __forceinline__ int k_tiles(const ExpertTile &) const { return g.k_tiles; }
  static constexpr bool kWarm = false;
  const mtk_mx_gemm_kargs &g;
  GroupSearch<BM> search;
  uint32_t row_b;
  __device__ __forceinline__ explicit MxTiles(const mtk_mx_gemm_kargs &g_)
      : g(g_), search(g_.row_start, g_.row_start ? g_.E : 0, g_.T, g_.tiles_n), row_b((uint32_t)mx_row_bytes(g_.k_tiles)) {
    if (!g.row_start) search.total = (g.T + BM - 1) / BM * g.tiles_n;
  }
  __device__ __forceinline__ int lda() const { return (int)(row_b >> 1); }
  __device__ __forceinline__ int ldb() const { return (int)(row_b >> 1); }
  __device__ __forceinline__ int ldc() const { return g.ldc; }
  __device__ __forceinline__ bool f32() const { return false; }
  __device__ __forceinline__ bool streamed() const { return false; }
  __device__ __forceinline__ size_t a_step() const { return (size_t)g.T * 8; }
  __device__ __forceinline__ size_t b_step() const { return (size_t)g.E * (size_t)g.N * 8; }
  __device__ __forceinline__ ExpertTile get(int i) const {
    ExpertTile t{};
    GroupTile gt;
    int half;
    if (g.row_start) {
      gt = search.get(i, half);
    } else {
      const group_place place = nth_tile<BM>(i, search.total);
      half = place.half;
      gt.t = place.tile;
      gt.e = gt.t < 0 ? -1 : 0;
      gt.first = 0;
      gt.rows = g.T;
      gt.blocks = (g.T + BM - 1) / BM;
    }
    if (gt.e < 0) return t;
    const TileAt at = tile_at<BM, BN>(gt.t, gt.blocks, g.tiles_n);
    const int m0 = at.m0 + half_first<BM>(half);
    const int64_t row = gt.first + m0, col = (int64_t)gt.e * g.N + at.n0;
    t.rows = half_rows<BM>(half, gt.rows - m0);
    t.there = t.rows > 0;
    if (!t.there) return t;
    t.cols = min(g.N - at.n0, BN);
    t.a = (const char *)g.A + row * (int64_t)row_b;
    t.b = (const char *)g.B + col * (int64_t)row_b;
    t.sa = (const char *)g.a_scales + row * 8;
    t.sb = (const char *)g.b_scales + col * 8;
    t.a_bytes = (uint32_t)t.rows * row_b;
    t.b_bytes = (uint32_t)t.cols * row_b;
    t.c = (char *)g.C + ((size_t)row * (size_t)g.ldc + (size_t)at.n0) * 2;
    t.bias = g.has_bias ? (const uint16_t *)g.bias + col : nullptr;
    t.turn = g.turns.on ? group_turn(group_turn_place(gt.e, at.n0 / BN, g.turns), whole()) : 0;
    return t;
  }
};

// ---------------------------------------------------------------- the pipeline

// One of two values (an expression of two fields would choose between their addresses, and put both structures into memory).
template <class T>
__device__ __forceinline__ T pick(bool first, T x, T y) {
  return first ? x : y;
}

template <class EL, int BM, int BN, int WM, int WN, class AOP, class BOP, class TILES>
__device__ __forceinline__ void expert_tiles(const TILES &tiles) {
  constexpr int DT = EL::DT;
  constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  constexpr int kCodes = AOP::kBytes + BOP::kBytes, kStage = kCodes + (EL::kScales ? (BM + BN) * 8 : 0);
  constexpr int PA = AOP::kLoads, PB = BOP::kLoads, kLoads = PA + PB + (EL::kScales ? 1 : 0);
  constexpr int kScaleLoads = (BM + BN) / 128;  // of all wavefronts
  static_assert(!EL::kScales || (kScaleLoads <= NW && BM % 128 == 0 && BN % 128 == 0), "a wavefront has one load of scales at most");
  static_assert(WTN == 64 && TM % 2 == 0, "epilogue rows of 128 bytes, halves of a wavefront's rows");
  constexpr bool kWarm = TILES::kWarm;
  constexpr int kSpare = EL::kScales || kWarm ? 1024 : 0, kPark = 2 * kStage + kSpare;  // behind the stages: [wave][16 rows][128 bytes]
  static_assert(kPark + NW * 2048 <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) char smem[kPark + NW * 2048];

  ExpertTile cur = tiles.get(0);
  if (!cur.there) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / WN, wave_n = wave % WN;
  const AOP opa(wave, lane, (uint32_t)tiles.lda() * 2u);
  const BOP opb(wave, lane, (uint32_t)tiles.ldb() * 2u);
  const uint32_t lds = lds_addr(smem);

  // scales: wavefront w loads those of rows 128 w .. 128 w + 127 of A, then of B; the others load zeros to the bytes behind the
  // stages (a branch in the loop would let the compiler move its MFMAs past the loads)
  const bool scales_a = wave < BM / 128, scales = wave < kScaleLoads;
  const int at_s = scales ? kCodes + wave * 1024 : 2 * kStage, next_s = scales ? kStage : 0;
  const uint32_t off_s = (uint32_t)(scales_a ? wave : wave - BM / 128) * 1024u + 16u * (uint32_t)lane;

  // The buffers of one K-tile's loads: K-tile k of t, or k - n of u where t has no more.
  struct Source {
    rsrc_t a, b, s;
  };
  auto source = [&](const ExpertTile &t, const ExpertTile &u, int n, int k) {
    const bool own = k < n;
    k = own ? k : k - n;
    if constexpr (TILES::kTurned) k = group_turned(k, pick(own, t.turn, u.turn), tiles.whole());
    const int K = pick(own, tiles.K(t), tiles.K(u));
    const bool there = k < pick(own, tiles.k_tiles(t), u.there ? tiles.k_tiles(u) : 0);
    Source r;
    r.a = AOP::at(pick(own, t.a, u.a), pick(own, t.a_bytes, u.a_bytes), tiles.lda(), K, k, there);
    r.b = BOP::at(pick(own, t.b, u.b), pick(own, t.b_bytes, u.b_bytes), tiles.ldb(), K, k, there);
    if constexpr (EL::kScales) {
      const char *const p = pick(scales_a, pick(own, t.sa, u.sa), pick(own, t.sb, u.sb));
      const int rows = pick(scales_a, pick(own, t.rows, u.rows), pick(own, t.cols, u.cols));
      r.s = make_rsrc(p + (size_t)k * (scales_a ? tiles.a_step() : tiles.b_step()), there && scales ? (uint32_t)rows * 8u : 0u);
    }
    return r;
  };
  auto issue = [&](auto q_c, const Source &r, int st) {  // load q of this wavefront into stage st
    constexpr int q = decltype(q_c)::value;
    char *const at = smem + st * kStage;
    if constexpr (q < PA)
      lds_direct16(r.a, at + (wave * PA + q) * 1024, opa.off[q]);
    else if constexpr (q < PA + PB)
      lds_direct16(r.b, at + AOP::kBytes + (wave * PB + q - PA) * 1024, opb.off[q - PA]);
    else
      lds_direct16(r.s, smem + at_s + st * next_s, off_s);
  };

  f32x16 acc[TM][TN];
  u32x4 fa[2][TM] = {}, fb[2][TN] = {};
  uint32_t sa[TM] = {}, sb[TN] = {}, na[TM] = {}, nb[TN] = {};  // this K-tile's scales, and the next one's
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
  };
  // read r of the fragments of k-step ks: B's, then A's of the first NI blocks
  auto read_frag = [&](auto ks_c, auto r_c, auto ni_c, int st) {
    constexpr int ks = decltype(ks_c)::value, r = decltype(r_c)::value;
    const uint32_t at = lds + (uint32_t)(st * kStage);
    if constexpr (r < TN)
      fb[ks & 1][r] = BOP::template frag<ks>(at + AOP::kBytes, wave_n * TN + r, lane);
    else if constexpr (r < TN + decltype(ni_c)::value)
      fa[ks & 1][r - TN] = AOP::template frag<ks>(at, wave_m * TM + r - TN, lane);
  };
  auto read_scales = [&](int st) {
    if constexpr (EL::kScales) {
      const uint32_t s = lds + (uint32_t)(st * kStage + kCodes + 8 * (lane & 31) + 4 * (lane >> 5));
      static_for<0, TN>([&](auto j) { nb[j] = ds_read_b32_at<256 * j>(s + (uint32_t)(BM + wave_n * WTN) * 8u); });
      static_for<0, TM>([&](auto i) { na[i] = ds_read_b32_at<256 * i>(s + (uint32_t)(wave_m * WTM) * 8u); });
    }
  };
  // All LDS reads have landed: what they fill may be used from here on, and copied by the compiler.
  auto landed = [&]() {
    frag_wait<0>(fa[0], fb[0]);
    if constexpr (EL::kScales) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        asm volatile("" : "+v"(na[i]));
        sa[i] = na[i];
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        asm volatile("" : "+v"(nb[j]));
        sb[j] = nb[j];
      }
    }
  };

  // One K-tile of stage st, whose row blocks from NI on are not multiplied, and the loads of next() into that stage.
  // Where tiles are turned next() is computed behind a step's first MFMAs, so that the turn costs nothing: one group of 8192 rows of 4096 x
  // 4096, zeros, 163 -> 151 us (random data 214.3 -> 214.4). Gradients lose by that: 8192 rows over 16 groups 304 -> 310.
  auto ktile = [&](auto ni_c, int st, auto next) {
    constexpr int NI = decltype(ni_c)::value;
    Source src;
    if constexpr (!TILES::kTurned) src = next();
    constexpr int kReads = (TM + TN + 1) / 2, kLoadsPer = (kLoads + TM - 1) / TM;
    static_for<0, 4>([&](auto k_c) {
      constexpr int ks = decltype(k_c)::value;
      if constexpr (ks > 0) frag_wait<0>(fa[ks & 1], fb[ks & 1]);
      if constexpr (ks == 3) {
        vm_wait<0>();
        __builtin_amdgcn_s_barrier();
      }
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, TM>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        if constexpr (i < NI) {
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = EL::template mfma<ks>(fa[ks & 1][i], fb[ks & 1][j], acc[i][j], sa[i], sb[j]);
        }
        if constexpr (i < 2 && NI > 0)
          static_for<i * kReads, (i + 1) * kReads>(
              [&](auto r) { read_frag(std::integral_constant<int, (ks + 1) & 3>{}, r, ni_c, ks == 3 ? st ^ 1 : st); });
        if constexpr (ks == 3) {
          if constexpr (i == 1 && NI > 0) read_scales(st ^ 1);
          static_for<i * kLoadsPer, ((i + 1) * kLoadsPer < kLoads ? (i + 1) * kLoadsPer : kLoads)>([&](auto q) { issue(q, src, st); });
        }
        if constexpr (TILES::kTurned && ks == 1 && i == 0) src = next();
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    landed();  // nothing is in flight at the loop's back edge
  };

  // ---- a tile's outputs: lane l, register r of a 32x32 block holds row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32. Neighbours
  // swap one value of each register pair, so that every lane has two columns of one row.
  auto store = [&](const ExpertTile &t) {
    int le = lane_id();
    asm volatile("" : "+v"(le));
    const bool odd = le & 1;
    const int col_l = (le & 31) & ~1, row_l = 4 * (le >> 5) + (odd ? 1 : 0);
    auto pair = [&](float x0, float x1, float &lo, float &hi) {
      const float send = odd ? x0 : x1;
      const float recv = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, send), 0xB1, 0xF, 0xF, false));
      lo = odd ? recv : x0;
      hi = odd ? x1 : recv;
    };
    const int rows = t.rows - wave_m * WTM, cols = t.cols - wave_n * WTN;
    if (rows <= 0 || cols <= 0) return;
    const int ldc = tiles.ldc();
    const size_t at = (size_t)(wave_m * WTM) * (size_t)ldc + (size_t)(wave_n * WTN);
    if (tiles.f32()) {
      float *C = (float *)t.c + at;
      // Past the caches where rows are whole halves of lines: 7183 rows, 128 groups of 6640 x 128 119 -> 85 us; rows of other lengths
      // leave parts of lines for the L2 to join: 471 rows, 128 of 256 x 2616 190 -> 119 through it.
      const bool streamed = (ldc & 15) == 0 && ((uintptr_t)C & 63) == 0;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int col = col_l + 32 * j;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            float lo, hi;
            pair(acc[i][j][r], acc[i][j][r + 1], lo, hi);
            const int row = row_l + 32 * i + 8 * (r >> 2) + (r & 3);
            if (row >= rows) continue;
            float *p = C + (size_t)row * (size_t)ldc + col;
            if (col + 1 < cols) {
              if (streamed)
                __builtin_nontemporal_store(f32x2{lo, hi}, (f32x2 *)p);
              else
                ((Pair *)p)->v = f32x2{lo, hi};
            } else if (col < cols) {
              *p = lo;
            }
          }
      }
      return;
    }
    float bv[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int own = col_l + 32 * j + (odd ? 1 : 0);  // the column that this lane's accumulators belong to
      bv[j] = t.bias && own < cols ? from_bits<DT>(t.bias[wave_n * WTN + own]) : 0.0f;
    }
    uint16_t *C = (uint16_t *)t.c + at;
    const bool streamed = tiles.streamed() && (ldc & 31) == 0 && ((uintptr_t)C & 63) == 0;
    const uint32_t park = lds + (uint32_t)(kPark + wave * 2048);
    // The chunk swizzle puts the four rows that one write touches on different banks. Reads and writes of a wavefront are done in
    // order; inline asm, as the compiler would make them wait for the loads in flight.
    auto swz = [](int rr) { return 4 * ((rr >> 2) & 1); };
#pragma unroll
    for (int p = 0; p < 2 * TM; ++p) {  // 16 rows at a time
      const int i = p >> 1, half = p & 1;
      if (16 * p >= rows) break;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int cc = col_l + 32 * j;
#pragma unroll
        for (int r = 8 * half; r < 8 * half + 8; r += 2) {
          float lo, hi;
          pair(acc[i][j][r] + bv[j], acc[i][j][r + 1] + bv[j], lo, hi);
          const int rr = row_l + 8 * ((r >> 2) & 1) + (r & 3);
          const uint32_t v = pack2<DT>(lo, hi);
          asm volatile("ds_write_b32 %0, %1" ::"v"(park + (uint32_t)(rr * 128 + (((cc >> 3) ^ swz(rr)) << 4) + (cc & 7) * 2)), "v"(v) : "memory");
        }
      }
      u32x4 v[2];
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int rr = 8 * it + (le >> 3), ch = le & 7;
        v[it] = lds_rd128(park + (uint32_t)(rr * 128 + ((ch ^ swz(rr)) << 4)));
      }
      lgkm_wait0(v);
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int row = 16 * p + 8 * it + (le >> 3), c8 = 8 * (le & 7);
        if (row < rows) {
          uint16_t *dst = C + (size_t)row * (size_t)ldc + c8;
          if (c8 + 8 <= cols) {
            if (streamed)
              __builtin_nontemporal_store(v[it], (u32x4 *)dst);
            else
              ((Chunk *)dst)->v = v[it];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t w = v[it][e >> 1];
              if (c8 + e < cols) dst[e] = (uint16_t)((e & 1) ? (w >> 16) : (w & 0xffffu));
            }
          }
        }
      }
    }
  };

  // The last K-tile of rows whose K is no multiple of 64 holds what follows in memory: it has landed in stage st, and here a
  // thread per row makes zeros of it. (Both operands': a NaN times zero is none.)
  auto cut = [&](int st, int k) {
    constexpr int kA = AOP::kMasked ? BM : 0, kRows = kA + (BOP::kMasked ? BN : 0);
    static_assert(kRows <= 64 * NW, "a thread per row");
    if ((int)threadIdx.x < kRows) {
      const int row = (int)threadIdx.x < kA ? (int)threadIdx.x : (int)threadIdx.x - kA;
      const uint32_t at = lds + (uint32_t)(st * kStage + ((int)threadIdx.x < kA ? 0 : AOP::kBytes));
      for (int c = k >> 3; c < 8; ++c) {
        const uint32_t p = at + lds_off(row, c);
        u32x4 v[1] = {lds_rd128(p)};
        lgkm_wait0(v);
        lds_wr128(p, keep_halves(v[0], k - 8 * c));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
  };

  {
    const Source s0 = source(cur, cur, 2, 0), s1 = source(cur, cur, 2, 1);
    static_for<0, kLoads>([&](auto q) { issue(q, s0, 0); });
    static_for<0, kLoads>([&](auto q) { issue(q, s1, 1); });
    vm_wait<kLoads>();  // the first K-tile's
    __builtin_amdgcn_s_barrier();
  }
  int st = 0;
#pragma unroll 1
  for (int i = 0;; ++i) {
    const ExpertTile next = tiles.get(i + 1);
    const int n = max(tiles.k_tiles(cur), 2);
    clear();
    const int blocks = cur.cols > wave_n * WTN ? (cur.rows - wave_m * WTM + 31) >> 5 : 0;
    auto run = [&](auto ni_c) {
      int k = 0;
      auto first = [&]() {
        if constexpr (decltype(ni_c)::value > 0) {
          static_for<0, TM + TN>([&](auto r) { read_frag(std::integral_constant<int, 0>{}, r, ni_c, st); });
          read_scales(st);
        }
        landed();
      };
      first();
      // K-tile k of this tile, and the loads of the one after the next, which may be the next tile's
      auto upto = [&](int stop) {
#pragma unroll 1
        for (; k < stop; ++k) {
          ktile(ni_c, st, [&]() { return source(cur, next, n, k + 2); });
          st ^= 1;
        }
      };
      if constexpr (AOP::kMasked || BOP::kMasked) {
#pragma unroll 1
        for (int stop = (tiles.K(cur) & 63) != 0 ? tiles.k_tiles(cur) - 1 : n;; stop = n) {
          upto(stop);
          if (stop == n) break;
          cut(st, tiles.K(cur) & 63);
          first();
        }
      } else if constexpr (kWarm) {
#pragma unroll 1
        for (int stop = next.there && next.e != cur.e ? n - 2 : n;; stop = n) {
          upto(stop);
          if (stop == n) break;
          lds_direct16(tiles.warm(wave), smem + 2 * kStage, tiles.warm_off(next, wave, lane));
        }
      } else {
        upto(n);
      }
    };
    if (blocks > TM / 2)
      run(std::integral_constant<int, TM>{});
    else if (blocks > 0)
      run(std::integral_constant<int, TM / 2>{});
    else
      run(std::integral_constant<int, 0>{});
    store(cur);
    if (!next.there) break;
    cur = next;
  }
  wait_vmem();  // no load into LDS is in flight when the workgroup ends
}

}  // namespace mtk
