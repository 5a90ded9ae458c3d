// Attention over a paged key/value cache in few bits (fp4 or fp8 blocks of 32 dims with a power-of-two scale,
// kv_cache.h), ragged batch, grouped heads: few rows per sequence (a decode step, drafted tokens).
//
//   O[i][h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(q_i . k_j / sqrt(D)),  j <= position of row i (causal)
//
// with k_j, v_j the cached values. One pass over the keys with a running exponent offset and sum per row (fp32).
//   * The wavefronts of a workgroup (4, 8 or 16) take tiles of 32 or 64 keys in turn for the same 16 NR (row, query head) pairs
//     of a K/V head. Where a sequence's pairs are few enough for one workgroup each (runtime: plan_kv_attn), that is all;
//     else the steps of all pairs lie on a line that persistent workgroups share evenly (kv_cache.h), found on the device
//     from the lengths, so that a captured launch serves any lengths. fp8, 16 x 8192 ragged positions: equal splits of each
//     sequence 68 us, of all of them 55.
//   * K: a lane has the codes of one key and a quarter of the head's dims: exactly an operand of the 16x16x32
//     MFMA (the dims may be summed in any order, Q is loaded in the same one). They go from the load through
//     v_cvt_scalef32_pk (two codes and their scale per instruction, exact) into S^T = K Q^T without LDS.
//   * S^T leaves each lane with 4 keys of one row per 16 keys, which is the operand layout of P^T in
//     O^T = V^T P^T. V^T needs 8 keys of one dim per lane: V is converted the same way, written to the
//     wavefront's own LDS tile and read back transposed (ds_read_b64_tr_b16).
//   * P is rounded to the 16-bit type for the MFMA (off by up to 2^-8 or 2^-11 of its value, averaged over the keys; f16: or by
//     2^-32 of the row's largest weight, kv_join.hpp); scores, offsets and sums stay in fp32.
//   * Keys past the length have their V codes zeroed (a page's unused rows may hold anything); a NaN block's V is
//     zeroed too and its dims set to NaN only for the rows that see the key, so that nothing masked reaches O.
//
// Bound: HBM where there is much to read, else latency. A wavefront's loads of the next tile are issued as its registers
// fall free (K and scales before the softmax, V after its codes are staged); nothing spills, for scratch traffic cost more
// than a third wavefront per SIMD won (fp8, 128 dims: 3 per SIMD 49.7 us, 4 with spills 58.7). The next tile's loads are
// behind a branch: issued always, with an empty range past the last one, 33.0 us instead of 31.7. Loads that bypass the caches: 5 % faster on one long
// sequence, 12 to 18 % slower where sequences share pages. Scales as whole words: 64 dims 41.4 -> 36.5 us.
// Measured, three sets of operands in turn, tables that end with the longest sequence (figures of a profiler's trace, 1 to 3 % above
// those of a stream of calls; sets of 900 MB in turn, past the last-level cache: 1 to 10 % more): fp4, 8 K/V heads of 128 dims, 4
// query heads each, first kernel and join: 1 x 131071 positions 32.2 + 7.2 us
// (4.5 TB/s in the first), 64 x 6000 82 + 7 (5.1 TB/s), 32 x 4096 ragged 22.4, 1 x 1000 9.0 (0.8 to find its work, 1.6 for
// the first bytes, 2 tiles of 1.1, 2.4 for the sum over 16 wavefronts, the launch); 64-dim heads without groups, 64 x 2048:
// 29.4; fp8 16 x 8192: 50.4 + 4.9 (4.8 TB/s).
#include "kv_join.hpp"

namespace mtk {

constexpr int kWindow = 56;       // table entries between the starts of two windows (below)

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarters_max(float x) {
  x = half_max(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return __builtin_elementwise_maximum(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float quarters_sum(float x) {
  x = half_sum(x);
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}

template <int DT, int FMT, int DP, int NR, int KB, int W>
__device__ __forceinline__ void kv_attend(const mtk_kv_attn_kargs &a) {
  constexpr int kRows = 16 * NR, kKvTile = 16 * KB, kKvStep = kKvTile * W;
  constexpr int kFr = DP / 32;                // operands of 8 dims per lane and key
  constexpr int kW8 = kWords8<FMT>;
  constexpr int kRaw = kFr * kW8;             // words of codes per lane and key
  constexpr int kSc = DP == 256 ? 2 : 1;      // scales per lane and key
  constexpr int kKb = KB;                     // 16-key blocks per tile
  constexpr int kDb = DP / 16;                // 16-dim blocks of O
  constexpr int kVRowB = 2 * DP;
  constexpr int kWaveB = 32 * kVRowB;         // V is staged 32 keys at a time
  constexpr int kPitch = DP + 4;              // floats per parked row
  constexpr int kParkB = 16 * kPitch * 4;
  __shared__ __attribute__((aligned(1024))) char smem[W * (kWaveB > kParkB ? kWaveB : kParkB)];
  __shared__ float sm_m[W][16], sm_l[W][16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, j = lane >> 4;
  const int G = a.G;

  __shared__ int sm_window[W == 16 ? 1 : W][128];
  __shared__ int sm_line[W == 16 ? 1 : W][kLineWords];  // 16 wavefronts: pairs are whole
  KvLine<kRows, kKvStep> line(a, lane, sm_line[W == 16 ? 0 : wave]);
  int wg = 0, line_from = 0, line_to = 0;
  KvSegment seg;
  const bool whole = W == 16 || a.whole;
  if (whole) {  // a workgroup for each pair, by its number: nothing to look up
    seg.b = kv_div(blockIdx.x, a.H_kv);
    seg.hk = blockIdx.x - seg.b * a.H_kv;
    seg.rb = 0;
    seg.seq = load_seq(a, seg.b);
    const kv_share h = line.share_of(seg.seq);
    seg.from = seg.start = 0;
    seg.to = seg.steps = h.steps;
    if (h.blocks == 0) return;
  } else {
    line.lay();
    const int wgs = kv_div(line.total + line.cut.each - 1, line.cut.each);
    if ((int)blockIdx.x >= wgs) return;
    wg = xcd_remap(blockIdx.x, wgs);
    line_from = wg * line.cut.each;
    line_to = min(line.total, line_from + line.cut.each);
    seg = line.at(line_from, line_to);
    if (seg.b < 0) return;
  }

  // ---- this lane's place in 16 positions of codes and scales. Lanes of blocks past the head's last read the last
  // one: Q is zero there, and those dims of O are not stored.
  const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
  const uint64_t region = kv_region_bytes(FMT, a.blocks, a.page_shift), page_b = region * (uint64_t)a.H_kv;
  const int page_mask = (1 << a.page_shift) - 1;
  const uint32_t k_scales = (2 * row_b) << a.page_shift, v_codes = row_b << a.page_shift;
  const uint32_t v_scales = k_scales + ((uint32_t)a.blocks << a.page_shift);
  constexpr uint32_t kHalf = FMT == KV_FP4 ? 8 : 16;  // bytes of half a block
  uint32_t code_at[kSc], scale_at[kSc], scale_bit[kSc];  // scales are loaded as whole words
#pragma unroll
  for (int s = 0; s < kSc; ++s) {
    const int blk = min(DP == 64 ? j >> 1 : j + 4 * s, a.blocks - 1);
    code_at[s] = c * row_b + blk * 2 * kHalf + (DP == 64 ? (j & 1) * kHalf : 0u);
    scale_at[s] = (uint32_t)(c * a.blocks + blk) & ~3u;
    scale_bit[s] = 8 * ((uint32_t)(c * a.blocks + blk) & 3u);
  }
  struct Tile {
    uint32_t k[kKb][kRaw], v[kKb][kRaw], ks[kKb][kSc], vs[kKb][kSc];
    uint32_t bad = 0;  // 16-key blocks whose page is not one
  };

  // ---- what the loads of a segment need: its pages, as table entries that the lanes hold, 64 in a window and 64 in
  // the next window, which starts kWindow entries on, so that a tile lies in one of the two
  struct Source {
    const char *head;     // the K/V head's region of page 0
    const int32_t *table;
    uint32_t pages;       // entries below it are pages
    int last_block, e0, window, next_window;
    int key0, key_end, n_keys;  // this wavefront's first key, the segment's end, the keys that its rows see
  };
  auto source = [&](const KvSegment &g, bool windows) {
    Source x;
    const int rows = min(g.seq.rows, a.S_q) * G, r_last = min(g.rb * kRows + kRows, rows) - 1;
    const int64_t p_last = a.causal ? g.seq.pos0 + kv_div(r_last, G) : (int64_t)g.seq.keys - 1;
    x.n_keys = (int)max((int64_t)0, min((int64_t)g.seq.keys, p_last + 1));
    x.key_end = min(x.n_keys, g.to * kKvStep);
    x.key0 = g.from * kKvStep + wave * kKvTile;
    x.head = (const char *)a.cache + (uint64_t)(uint32_t)g.hk * region;
    x.table = a.table + (size_t)(uint32_t)g.b * (uint32_t)a.max_pages;
    x.pages = g.seq.bad ? 0u : (uint32_t)a.n_pages;
    x.last_block = (max(x.n_keys, 1) - 1) & ~15;
    x.e0 = x.key0 >> a.page_shift;
    if (windows) {
      x.window = x.table[min(x.e0 + lane, a.max_pages - 1)];
      x.next_window = x.table[min(x.e0 + kWindow + lane, a.max_pages - 1)];
    }
    return x;
  };
  // Where the blocks of a tile are. The range of the loads is the page's region.
  struct Place {
    rsrc_t r[kKb];
    uint32_t at[kKb];
  };
  auto locate = [&](Tile &t, Source &x, int key0) {
    if ((min(key0 + kKvTile - 16, x.last_block) >> a.page_shift) - x.e0 >= 64) {
      x.e0 += kWindow;
      x.window = x.next_window;
      x.next_window = x.table[min(x.e0 + kWindow + lane, a.max_pages - 1)];
    }
    t.bad = 0;
    Place p;
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb) {
      const int key = min(key0 + 16 * kb, x.last_block);  // blocks past the keys: any, they are masked
      uint32_t page = (uint32_t)__builtin_amdgcn_readlane(x.window, (key >> a.page_shift) - x.e0);
      if (page >= x.pages) {
        t.bad |= 1u << kb;
        page = 0;
      }
      p.r[kb] = make_rsrc(x.head + (uint64_t)page * page_b, (uint32_t)region);
      p.at[kb] = (uint32_t)(key & page_mask);
    }
    return p;
  };
  auto load_scales = [&](Tile &t, const Place &p) {
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
      for (int s = 0; s < kSc; ++s) {
        const uint32_t at = p.at[kb] * (uint32_t)a.blocks;
        t.ks[kb][s] = __builtin_amdgcn_raw_buffer_load_b32(p.r[kb], scale_at[s], k_scales + at, 0);
        t.vs[kb][s] = __builtin_amdgcn_raw_buffer_load_b32(p.r[kb], scale_at[s], v_scales + at, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Codes of K (which 0) or V (1) of blocks b0 to b1 - 1.
  auto load = [&](Tile &t, const Place &p, int which, int b0, int b1) {
#pragma unroll
    for (int kb = b0; kb < b1; ++kb)
#pragma unroll
      for (int s = 0; s < kSc; ++s) {
        constexpr int kN = kRaw / kSc;
        uint32_t *w = (which ? t.v[kb] : t.k[kb]) + s * kN;
        const uint32_t so = (which ? v_codes : 0u) + p.at[kb] * row_b;
        if constexpr (kN == 2) {
          const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(p.r[kb], code_at[s], so, 0);
          w[0] = x[0], w[1] = x[1];
        } else {
#pragma unroll
          for (int q = 0; q < kN / 4; ++q) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(p.r[kb], code_at[s] + 16 * q, so, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * q + i] = x[i];
          }
        }
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto load_tile = [&](Tile &t, Source &x, int key0) {
    const Place p = locate(t, x, key0);
    load_scales(t, p);
    load(t, p, 0, 0, kKb);
    load(t, p, 1, 0, kKb);
  };

  // V in 16 bits in LDS: chunk (8 dims) ch of key r at r * row + ((ch ^ swz(r)) * 16), swz(r) from bits 0 to 3 of r: the
  // chunks that 16 lanes write, and those that 32 lanes read transposed, lie in different banks. An operand's or a
  // block's chunk differs from the first one's in bits of its own, so that its address is the first one's with those
  // bits flipped (rows of 16 more keys: an offset).
  auto vswz = [](int r) {
    return DP == 64 ? (((r >> 1) & 3) << 1) | ((r >> 3) & 1) : ((r & 7) << 1) | ((r >> 3) & 1);
  };
  const int tr = 4 * j + (c >> 2);
  uint32_t v_put = (uint32_t)(wave * kWaveB + c * kVRowB + (((DP == 64 ? 2 * j : 4 * j) ^ vswz(c)) << 4));
  uint32_t v_get = (uint32_t)(wave * kWaveB + tr * kVRowB + ((((c & 3) >> 1) ^ vswz(tr)) << 4) + 8 * (c & 1));
  const float cl = a.scale_log2;

  // ---- Q, as the operand of S^T: row c of each 16, this lane's dims
  auto dim = [&](int f) { return DP == 64 ? 16 * j + 8 * f : 128 * (f >> 2) + 32 * j + 8 * (f & 3); };
  u32x4 qf[NR][kFr];
  int lim[NR];  // the last key that this lane's row sees
  auto load_q = [&](const KvSegment &g) {
    const int rows = min(g.seq.rows, a.S_q) * G;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = g.rb * kRows + 16 * n + c, i = kv_div(r, G);
      const int64_t pos = a.causal ? g.seq.pos0 + i : (int64_t)g.seq.keys - 1;
      lim[n] = r < rows && pos >= 0 ? (int)min(pos, (int64_t)g.seq.keys - 1) : -1;
      const uint16_t *q = (const uint16_t *)a.Q + (size_t)(g.seq.first + i) * a.ld_q + (size_t)(g.hk * G + r - i * G) * a.D;
#pragma unroll
      for (int f = 0; f < kFr; ++f) {
        qf[n][f] = u32x4{0u, 0u, 0u, 0u};
        if (r < rows && dim(f) < a.D) qf[n][f] = *(const u32x4 *)(q + dim(f));
      }
    }
  };

  Source src = source(seg, true);
  load_q(seg);
  Tile t;
  if (src.key0 < src.key_end) load_tile(t, src, src.key0);

  for (;;) {
    // the next segment's table entries, ahead of their use
    const bool more = !whole && !line.cut.padded && seg.start + seg.to < line_to;
    if (more) {
      const Source x = source(line.at(seg.start + seg.to, line_to), true);
      sm_window[wave][lane] = x.window;  // in LDS until then, for want of registers
      sm_window[wave][64 + lane] = x.next_window;
    }
    float m_off[NR], l_run[NR];
    f32x4 o[NR][kDb];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      m_off[n] = first_offset(lim[n] >= 0);
      l_run[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < kDb; ++d) o[n][d] = f32x4{};
    }
    const int n_keys = src.n_keys, key_end = src.key_end;
    // keys that every row of the workgroup sees
    const int64_t p_first = a.causal ? seg.seq.pos0 + kv_div(seg.rb * kRows, G) : (int64_t)seg.seq.keys - 1;
    const int all_see = (int)max((int64_t)0, min((int64_t)seg.seq.keys, p_first + 1));
#pragma unroll 1
  for (int key0 = src.key0; key0 < key_end; key0 += kKvStep) {
    asm volatile("" : "+v"(v_put), "+v"(v_get));  // the flips are done in the loop: their results would fill registers
    // ---- NaN blocks and pages that are none: bit k of kn (vn[s][q]) is key k of the tile
    uint64_t kn = 0, vn[kSc][4] = {};
    uint32_t ks[kKb][kSc], vs[kKb][kSc];  // the next tile's are loaded before this one's have been used
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
      for (int s = 0; s < kSc; ++s) {
        ks[kb][s] = __builtin_amdgcn_ubfe(t.ks[kb][s], scale_bit[s], 8);
        vs[kb][s] = __builtin_amdgcn_ubfe(t.vs[kb][s], scale_bit[s], 8);
      }
    uint32_t top = t.bad ? kNanScale : 0;
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
      for (int s = 0; s < kSc; ++s) top = max(top, max(ks[kb][s], vs[kb][s]));
    const bool rare = __any(top == kNanScale);
    if (rare) {
#pragma unroll
      for (int kb = 0; kb < kKb; ++kb) {
        const bool none = (t.bad >> kb) & 1;
#pragma unroll
        for (int s = 0; s < kSc; ++s) {
          const uint64_t x = none ? ~0ull : __ballot(ks[kb][s] == kNanScale), y = none ? ~0ull : __ballot(vs[kb][s] == kNanScale);
          kn |= ((x | x >> 16 | x >> 32 | x >> 48) & 0xffff) << (16 * kb);
#pragma unroll
          for (int q = 0; q < 4; ++q) vn[s][q] |= ((y >> (16 * q)) & 0xffff) << (16 * kb);
          if (none || ks[kb][s] == kNanScale) ks[kb][s] = 127;
          if (none || vs[kb][s] == kNanScale) {
            vs[kb][s] = 127;
#pragma unroll
            for (int i = 0; i < kRaw / kSc; ++i) t.v[kb][s * (kRaw / kSc) + i] = 0;
          }
        }
      }
    }
    if (key0 + kKvTile > n_keys) {  // rows of a page past the length may hold anything
#pragma unroll
      for (int kb = 0; kb < kKb; ++kb)
        if (key0 + 16 * kb + c >= n_keys) {
#pragma unroll
          for (int i = 0; i < kRaw; ++i) t.v[kb][i] = 0;
#pragma unroll
          for (int s = 0; s < kSc; ++s) vs[kb][s] = 127;
        }
    }

    // ---- S^T = K Q^T
    f32x4 s[NR][kKb];
#pragma unroll
    for (int kb = 0; kb < kKb; ++kb) {
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][kb] = f32x4{};
#pragma unroll
      for (int f = 0; f < kFr; ++f) {
        const u32x4 kf = values8<DT, FMT>(t.k[kb] + f * kW8, scale_of(ks[kb][kSc == 2 ? f >> 2 : 0]));
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][kb] = mfma16x16x32<DT>(kf, qf[n][f], s[n][kb]);
      }
    }
    // ---- V in 16 bits to LDS: chunk (8 dims) ch of key r at r * row + ((ch ^ vswz(r)) * 16)
    auto stage = [&](int h) {
#pragma unroll
      for (int kb = 2 * h; kb < 2 * h + 2; ++kb) {
#pragma unroll
        for (int f = 0; f < kFr; ++f)
          *(u32x4 *)(smem + ((v_put ^ (uint32_t)((f < 4 ? f : f + 12) << 4)) + 16 * (kb & 1) * kVRowB)) =
              values8<DT, FMT>(t.v[kb] + f * kW8, scale_of(vs[kb][kSc == 2 ? f >> 2 : 0]));
      }
      // the tile is this wavefront's own: its LDS accesses complete in order, only the compiler has to keep the
      // reads (of other lanes' chunks) behind the writes
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    // the next tile's loads, each as soon as its registers are free
    const bool ahead = key0 + kKvStep < key_end;
    Place place;
    if (ahead) {
      place = locate(t, src, key0 + kKvStep);
      load_scales(t, place);
      load(t, place, 0, 0, kKb);
    }
    stage(0);
    if (ahead) load(t, place, 1, 0, 2);
    const bool masked = key0 + kKvTile > all_see;

    // ---- softmax of the tile: this lane has keys 16 kb + 4 j + i of row c
    u32x4 pf[NR][kKb / 2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (rare) {
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb) {
          const uint32_t mine = (uint32_t)(kn >> (16 * kb)) >> (4 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][kb][i] = (mine >> i) & 1 ? __builtin_nanf("") : s[n][kb][i];
        }
      }
      if (masked) {
#pragma unroll
        for (int kb = 0; kb < kKb; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][kb][i] = key0 + 16 * kb + 4 * j + i <= lim[n] ? s[n][kb][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < kKb; ++kb) mx = vmax3(vmax3(mx, s[n][kb][0], s[n][kb][1]), s[n][kb][2], s[n][kb][3]);
      const float m_tile = quarters_max(mx) * cl;
      float alpha = 1.0f;
      if (m_tile - m_off[n] > kKvLift<DT> + kKvSlack) {  // a difference: exact where scores are far from zero
        alpha = __builtin_amdgcn_exp2f(m_off[n] - (m_tile - kKvLift<DT>));
        m_off[n] = m_tile - kKvLift<DT>;
      }
      const float moff = m_off[n] == -INFINITY ? 0.0f : m_off[n];
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int d = 0; d < kDb; ++d) o[n][d] *= alpha;
      }
      float sum = 0.0f;
#pragma unroll
      for (int h = 0; h < kKb / 2; ++h) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][2 * h + (i >> 2)][i & 3], cl, -moff));
          sum += p[i];
        }
        pf[n][h] = u32x4{pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
      }
      l_run[n] = __builtin_fmaf(l_run[n], alpha, sum);
    }

    // ---- O^T += V^T P^T: two transposed reads (keys 4 j .. + 3 of each 16) per 16 dims
#pragma unroll
    for (int h = 0; h < kKb / 2; ++h) {
      if (h > 0) {
        stage(h);
        if (ahead) load(t, place, 1, 2 * h, 2 * h + 2);
      }
#pragma unroll
      for (int d = 0; d < kDb; ++d) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const char *p = smem + ((v_get ^ (uint32_t)(d << 5)) + 16 * e * kVRowB);
          const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
          const u32x2 y = __builtin_bit_cast(u32x2, x);
          w[2 * e] = y.x;
          w[2 * e + 1] = y.y;
        }
        const u32x4 vf = u32x4{w[0], w[1], w[2], w[3]};
#pragma unroll
        for (int n = 0; n < NR; ++n) o[n][d] = mfma16x16x32<DT>(vf, pf[n][h], o[n][d]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (rare) {  // the dims of a NaN block, for the rows that see the key
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int seen = lim[n] - key0 + 1;
        const uint64_t vis = seen >= 64 ? ~0ull : seen <= 0 ? 0ull : (1ull << seen) - 1;
#pragma unroll
        for (int d = 0; d < kDb; ++d) {
          // 32-dim block d / 2: lane quarter (d / 2) & 3 of scale d / 8; DP 64: quarters 2 (d / 2), + 1
          const uint64_t nm = DP == 64 ? vn[0][(d >> 1) * 2] : vn[d >> 3][(d >> 1) & 3];
          if (nm & vis) o[n][d] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        }
      }
    }
  }

    // the next segment's first tile and Q are on their way while this one's sums are joined
    KvSegment next = seg;
    if (more) {
      next = line.at(seg.start + seg.to, line_to);
      src = source(next, false);
      src.window = sm_window[wave][lane];
      src.next_window = sm_window[wave][64 + lane];
      load_q(next);
      if (src.key0 < src.key_end) load_tile(t, src, src.key0);
    }

    // ---- the wavefronts' sums, 16 rows at a time, in wavefront order
    // lane numbers taken anew: what follows from them is not kept in registers over the loop
    const int lane2 = lane_id(), tid2 = 64 * wave + lane2, c2 = lane2 & 15, j2 = lane2 >> 4;
    const bool alone = seg.from == 0 && seg.to == seg.steps;
    const int rows = min(seg.seq.rows, a.S_q) * G;
    const size_t place = (size_t)wg * 2 + (seg.start + seg.from == line_from ? 0 : 1);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float l_tot = quarters_sum(l_run[n]);
      __syncthreads();  // the staging tiles, or the last rows, have been read
      if (j2 == 0) {
        sm_m[wave][c2] = m_off[n];
        sm_l[wave][c2] = l_tot;
      }
      float *park = (float *)smem + wave * (kParkB / 4);
#pragma unroll
      for (int d = 0; d < kDb; ++d) *(f32x4 *)(park + c2 * kPitch + 16 * d + 4 * j2) = o[n][d];
      __syncthreads();
      for (int it = tid2; it < 16 * (DP / 4); it += 64 * W) {
        const int rr = it / (DP / 4), d0 = 4 * (it % (DP / 4));
        const int r = seg.rb * kRows + 16 * n + rr;
        if (r >= rows) continue;
        KvPart sum;
#pragma unroll
        for (int w = 0; w < W; ++w) sum.m = fmaxf(sum.m, sm_m[w][rr]);
        const float m0 = sum.m == -INFINITY ? 0.0f : sum.m;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float m = sm_m[w][rr], f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m0);  // no keys
          sum.l = __builtin_fmaf(f, sm_l[w][rr], sum.l);
          const f32x4 x = *(const f32x4 *)((const float *)smem + w * (kParkB / 4) + rr * kPitch + d0);
          sum.x = f32x4{__builtin_fmaf(f, x.x, sum.x.x), __builtin_fmaf(f, x.y, sum.x.y), __builtin_fmaf(f, x.z, sum.x.z),
                        __builtin_fmaf(f, x.w, sum.x.w)};
        }
        if (alone) {
          const int i = kv_div(r, G);
          store_out<DT>(a, seg.seq.first + i, seg.hk * G + r - i * G, d0, sum);
        } else {
          const size_t at = place * kRows + 16 * n + rr;
          if (d0 < a.part_ld) *(f32x4 *)(a.part + at * a.part_ld + d0) = sum.x;
          if (d0 == 0) *(f32x2 *)(a.part_ml + 2 * at) = f32x2{sum.m, sum.l};
        }
      }
    }
    if (!more) break;
    seg = next;
    __syncthreads();  // the parked sums have been read
  }
}

}  // namespace mtk

using namespace mtk;

#define MTK_KV_ATTEND(NAME, DT, FMT, DP, NR, KB, W, EU)                                              \
  extern "C" __global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(EU, EU))) \
  NAME(const mtk_kv_attn_kargs a) { kv_attend<DT, FMT, DP, NR, KB, W>(a); }
#define MTK_KV_ATTEND_FMT(NAME, FMT, DP, NR, KB, W, EU)                                 \
  MTK_KV_ATTEND(mtk_kv_attend_##NAME##_d##DP##_r##NR##_f16, DT_F16, FMT, DP, NR, KB, W, EU)   \
  MTK_KV_ATTEND(mtk_kv_attend_##NAME##_d##DP##_r##NR##_bf16, DT_BF16, FMT, DP, NR, KB, W, EU)

// mtk_kv_attend_<format>_d<padded head dimension>_r<16-row blocks per workgroup>_<type>: 16-key blocks per tile,
// wavefronts per workgroup, wavefronts per SIMD as the registers allow. runtime: kv_kernel_shape.
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 64, 1, 4, 4, 4)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 64, 2, 4, 8, 2)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 64, 4, 2, 4, 2)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 128, 1, 2, 4, 4)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 128, 2, 2, 8, 2)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 128, 4, 2, 4, 1)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 256, 1, 2, 8, 2)
MTK_KV_ATTEND_FMT(fp4, KV_FP4, 256, 2, 2, 4, 1)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 64, 1, 4, 4, 3)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 64, 2, 4, 8, 2)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 64, 4, 2, 4, 2)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 128, 1, 2, 4, 3)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 128, 2, 2, 8, 2)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 128, 4, 2, 4, 1)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 256, 1, 2, 8, 2)
MTK_KV_ATTEND_FMT(fp8, KV_FP8, 256, 2, 2, 4, 1)
// ..._w16: 16 wavefronts, for few pairs of short sequences, where a tile's latency counts
#define MTK_KV_ATTEND_W16(NAME, FMT, DP, KB)                                            \
  MTK_KV_ATTEND(mtk_kv_attend_##NAME##_d##DP##_r1_w16_f16, DT_F16, FMT, DP, 1, KB, 16, 4)     \
  MTK_KV_ATTEND(mtk_kv_attend_##NAME##_d##DP##_r1_w16_bf16, DT_BF16, FMT, DP, 1, KB, 16, 4)
MTK_KV_ATTEND_W16(fp4, KV_FP4, 64, 2)
MTK_KV_ATTEND_W16(fp4, KV_FP4, 128, 2)
MTK_KV_ATTEND_W16(fp8, KV_FP8, 64, 2)
MTK_KV_ATTEND_W16(fp8, KV_FP8, 128, 2)

#define MTK_KV_JOIN(NAME, DT, PARTS)                                                                   \
  extern "C" __global__ void __launch_bounds__(kKvJoin) NAME(const mtk_kv_attn_kargs a) {             \
    __shared__ int sm_line[kKvJoin / 64][kLineWords];                                                 \
    kv_join<DT, PARTS>(a, blockIdx.x, gridDim.x, sm_line);                                            \
  }
MTK_KV_JOIN(mtk_kv_join_rows_f16, DT_F16, false)
MTK_KV_JOIN(mtk_kv_join_rows_bf16, DT_BF16, false)
MTK_KV_JOIN(mtk_kv_join_parts_f16, DT_F16, true)
MTK_KV_JOIN(mtk_kv_join_parts_bf16, DT_BF16, true)
