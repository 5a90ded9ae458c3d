// Products of rows in few bits: C = A B_e^T + bias_e, A and B in blocks of 32 e2m1 values with one power-of-two scale (mx.h),
// fp32 accumulate on the scaled MFMA, which multiplies the codes' values exactly.
#include "mx_device.hpp"

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

// BM x BN tiles, WM x WN wavefronts: the GEMM's scheme (tile_direct.hpp) on rows of 128 bytes per K-tile, which are 256 places
// here: direct-to-LDS loads into two stages, swizzled on the global side, 32x32 blocks of the scaled MFMA, which takes the cycles
// of the 16-bit one for four times the K. A K-tile's scales (8 bytes a row) come with it, as a run of bytes behind the codes.
// Fragments are read one k-step ahead into two buffers, all of a step's reads in its first two groups of MFMAs. The barrier stands
// before the last k-step: then every wavefront has read the stage, the next K-tile has landed in the other one, whose first
// fragments and scales are read during that step, and the loads of the K-tile after it go into the stage that is free.
template <int DT, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void mx_tile_gemm(const mtk_mx_gemm_kargs &g) {
  constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  constexpr int kCodes = (BM + BN) * 128, kStage = kCodes + (BM + BN) * 8;
  constexpr int PA = BM / (8 * NW), PB = BN / (8 * NW);  // 1 KB loads of a wavefront and K-tile
  constexpr int kScaleLoads = (BM + BN) / 128;           // of all wavefronts
  static_assert(kScaleLoads <= NW && BM % 128 == 0 && BN % 128 == 0, "a wavefront has one load of scales at most");
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage + 1024];

  const GroupTile gt = mx_tile<BM>(g);
  if (gt.e < 0) return;
  const TileAt at = tile_at<BM, BN>(gt.t, gt.blocks, g.tiles_n);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / WN, wave_n = wave % WN;
  const int rows = min(gt.rows - at.m0, BM), cols = min(g.N - at.n0, BN);
  const int first = gt.first + at.m0;
  const MxOperand A(g.A, g.a_scales, first, rows, g.T, g.k_tiles);
  const MxOperand B(g.B, g.b_scales, (int64_t)gt.e * g.N + at.n0, cols, (int64_t)g.E * g.N, g.k_tiles);
  const int last = g.k_tiles - 1;

  // load q of a wavefront: rows 8 b .. 8 b + 7 of the tile (b = wave * P + q), lane l the chunk that belongs at byte 16 l
  uint32_t off_a[PA], off_b[PB];
  const uint32_t cbase = (uint32_t)((lane & 7) ^ (lane >> 3));
#pragma unroll
  for (int q = 0; q < PA; ++q) off_a[q] = (uint32_t)(8 * (wave * PA + q) + (lane >> 3)) * A.row_b + 16u * (cbase ^ ((wave * PA + q) & 7));
#pragma unroll
  for (int q = 0; q < PB; ++q) off_b[q] = (uint32_t)(8 * (wave * PB + q) + (lane >> 3)) * B.row_b + 16u * (cbase ^ ((wave * PB + q) & 7));
  // scales: wavefront w loads those of rows 128 w .. 128 w + 127 of A, then of B; the others load zeros to the bytes behind the
  // stages (a branch in the loop would let the compiler move its MFMAs past the loads)
  const bool scales_a = wave < BM / 128, scales = wave < kScaleLoads;
  const rsrc_t rs = scales_a ? A.scales : scales ? B.scales : make_rsrc(g.A, 0);
  const int at_s = scales ? kCodes + wave * 1024 : 2 * kStage, next_s = scales ? kStage : 0;
  const uint32_t off_s = (uint32_t)(scales_a ? wave : wave - BM / 128) * 1024u + 16u * (uint32_t)lane, step_s = scales_a ? A.tile_s : B.tile_s;
  auto issue = [&](auto q_c, int s, int kt) {  // load q of K-tile kt into stage s
    char *const st = smem + s * kStage;
    constexpr int q = decltype(q_c)::value;
    if constexpr (q < PA)
      lds_direct16(A.codes, st + (wave * PA + q) * 1024, off_a[q] + (uint32_t)kt * 128u);
    else if constexpr (q < PA + PB)
      lds_direct16(B.codes, st + BM * 128 + (wave * PB + q - PA) * 1024, off_b[q - PA] + (uint32_t)kt * 128u);
    else
      lds_direct16(rs, smem + at_s + s * next_s, off_s + (uint32_t)kt * step_s);
  };
  constexpr int kLoads = PA + PB + 1;

  // this lane's chunk at k-step ks of the 32-row block at row blk: 4 * (lane / 32) + ks, so that the scale word of a lane
  // has its four steps' bytes in order
  const int t0 = (lane & 7) ^ ((lane >> 3) & 3) ^ (4 * (lane >> 5));
  auto frag_at = [&](int blk, int ks) {
    return (uint32_t)(blk * 128 + (lane & 31) * 128 + ((t0 ^ ks ^ (4 * ((blk >> 5) & 1))) << 4));
  };
  const uint32_t scale_at = 8u * (uint32_t)(lane & 31) + 4u * (uint32_t)(lane >> 5);

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
  u32x4 fa[2][TM], fb[2][TN];
  uint32_t sa[TM], sb[TN], na[TM], nb[TN];  // this K-tile's scales, and the next one's
  // read r of the fragments of k-step ks: B's, then A's
  auto read_frag = [&](auto ks_c, auto r_c, const char *st) {
    constexpr int ks = decltype(ks_c)::value, r = decltype(r_c)::value;
    if constexpr (r < TN)
      fb[ks & 1][r] = ds_read_b128_at<0>(lds_addr(st) + BM * 128 + frag_at(wave_n * WTN + 32 * r, ks));
    else if constexpr (r < TN + TM)
      fa[ks & 1][r - TN] = ds_read_b128_at<0>(lds_addr(st) + frag_at(wave_m * WTM + 32 * (r - TN), ks));
  };
  auto read_scales = [&](const char *st) {
    const uint32_t s = lds_addr(st) + kCodes + scale_at;
    static_for<0, TN>([&](auto j) { nb[j] = ds_read_b32_at<256 * j>(s + (uint32_t)(BM + wave_n * WTN) * 8u); });
    static_for<0, TM>([&](auto i) { na[i] = ds_read_b32_at<256 * i>(s + (uint32_t)(wave_m * WTM) * 8u); });
  };
  auto take_scales = [&]() {  // after the wait for their reads
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
  };

  static_for<0, kLoads>([&](auto q) { issue(q, 0, 0); });
  static_for<0, kLoads>([&](auto q) { issue(q, 1, min(1, last)); });
  vm_wait<kLoads>();  // the first K-tile's
  __builtin_amdgcn_s_barrier();
  static_for<0, TM + TN>([&](auto r) { read_frag(std::integral_constant<int, 0>{}, r, smem); });
  read_scales(smem);
  // nothing is in flight where the compiler may copy registers into the loop's
  frag_wait<0>(fa[0], fb[0]);
  take_scales();

  constexpr int kReadGroups = TM > 1 ? 2 : 1;
  constexpr int kReads = (TM + TN + kReadGroups - 1) / kReadGroups, kLoadsPer = (kLoads + TM - 1) / TM;
#pragma unroll 1
  for (int kt = 0; kt <= last; ++kt) {
    char *const sc = smem + (kt & 1) * kStage;
    const char *const sn = smem + ((kt & 1) ^ 1) * kStage;
    const int kn = min(kt + 2, last);  // past the end the last K-tile again, never computed
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
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma_mx32<ks>(fa[ks & 1][i], fb[ks & 1][j], acc[i][j], sa[i], sb[j]);
        if constexpr (i < kReadGroups)
          static_for<i * kReads, (i + 1) * kReads>([&](auto r) { read_frag(std::integral_constant<int, (ks + 1) & 3>{}, r, ks == 3 ? sn : sc); });
        if constexpr (ks == 3) {
          if constexpr (i == kReadGroups - 1) read_scales(sn);
          static_for<i * kLoadsPer, ((i + 1) * kLoadsPer < kLoads ? (i + 1) * kLoadsPer : kLoads)>([&](auto q) { issue(q, kt & 1, kn); });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    // the next K-tile's first fragments and scales: nothing is in flight at the loop's back edge either
    frag_wait<0>(fa[0], fb[0]);
    take_scales();
  }

  // ---- epilogue as the GEMM's: the tile through LDS, so that a store instruction writes whole row segments of 16 bytes per lane
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
  constexpr int kRowB = WTN * 2, kChunks = kRowB / 16, kRowsPer = 64 / kChunks;
  static_assert(kChunks == 8 && NW * WTM * kRowB <= 2 * kStage, "C tile fits the LDS stages");
  auto swz = [](int rr) { return 4 * ((rr >> 2) & 1); };
  wait_vmem();
  __syncthreads();  // every wave is done reading, no load is in flight
  char *const ct = smem + wave * (WTM * kRowB);
  const uint16_t *bias = (const uint16_t *)g.bias + (size_t)gt.e * (size_t)g.N + at.n0;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int cc = col_l + 32 * j, own = wave_n * WTN + cc + (odd ? 1 : 0);
    const float bv = g.has_bias && own < cols ? from_bits<DT>(bias[own]) : 0.0f;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float lo, hi;
        pair(acc[i][j][r] + bv, acc[i][j][r + 1] + bv, lo, hi);
        const int rr = row_l + 32 * i + 8 * (r >> 2) + (r & 3);
        *(uint32_t *)(ct + rr * kRowB + (((cc >> 3) ^ swz(rr)) << 4) + (cc & 7) * 2) = pack2<DT>(lo, hi);
      }
  }
  uint16_t *C = (uint16_t *)g.C + (size_t)(first + wave_m * WTM) * (size_t)g.ldc + at.n0 + wave_n * WTN;
  const bool v16 = (g.ldc & 7) == 0 && ((uintptr_t)g.C & 15) == 0;
  const int rows_w = rows - wave_m * WTM, cols_w = cols - wave_n * WTN;
#pragma unroll 4
  for (int it = 0; it < WTM / kRowsPer; ++it) {
    const int rr = it * kRowsPer + le / kChunks, ch = le % kChunks;
    const u32x4 v = *(const u32x4 *)(ct + rr * kRowB + ((ch ^ swz(rr)) << 4));
    if (rr < rows_w) {
      uint16_t *dst = C + (size_t)rr * (size_t)g.ldc + 8 * ch;
      if (v16 && 8 * ch + 8 <= cols_w) {
        *(u32x4 *)dst = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = v[e >> 1];
          if (8 * ch + e < cols_w) dst[e] = (uint16_t)((e & 1) ? (w >> 16) : (w & 0xffffu));
        }
      }
    }
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
    mx_tile_gemm<DT, 256, 256, 2, 4>(g);                                                                         \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) mtk_mx_gemm_##NAME##_128(const mtk_mx_gemm_kargs g) {        \
    mx_tile_gemm<DT, 128, 128, 2, 2>(g);                                                                         \
  }
MTK_MX_GEMM(f16, DT_F16)
MTK_MX_GEMM(bf16, DT_BF16)
