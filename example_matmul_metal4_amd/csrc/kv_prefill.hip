// Attention over a paged key/value cache in few bits (kv_cache.h) for sequences with many new rows (a prompt's chunk):
// O = softmax(Q K^T / sqrt(D)) V as in kv_attention.hip, but the wavefronts of a workgroup split the rows.
//
//   * A workgroup has 128 (row, query head) pairs of one K/V head, each of its 4 wavefronts 32 of them, and walks the
//     keys in tiles of 64. K and V are converted once per workgroup: each thread has a block of 32 dims of one key of
//     both, loaded two or three tiles ahead, converted by v_cvt_scalef32_pk and written to LDS, two tiles each.
//   * S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMA, as the 128-query kernel of attention.hpp: a lane has one row of
//     the scores, K's rows are fed in the order that leaves P^T in the operand layout of the second product, V^T is
//     read by transposed LDS reads; the products of tile t + 1's scores alternate with the exponentials of tile t, the
//     second product with the maxima of tile t + 1.
//   * Grouped heads share a K/V head's tiles: 128 pairs are 128 / G queries.
//   * Keys past the length have their V codes zeroed, NaN blocks are zeroed in V and set to NaN for the rows that see
//     them, as in kv_attention.hip; bit masks of such keys lie in LDS beside the tiles.
//   * Few row blocks: the keys are split over workgroups (kv_cache.h), whose partial sums kv_join adds.
//
// Bound by the matrix units and the VALU beside them (the exponentials, and the conversions of a tile, shared by 128 pairs):
// 2048 rows of 32 heads of 128 dims behind 6144 positions 247 us with the launch before it, 0.97 PFLOP/s (262 where the card
// clocks lower, 269 to 300 under a profiler; fp8 257; 1024 rows of 256 dims 418, at half the rate with one workgroup per CU), where the 16-bit kernel of attention.hpp reaches 0.93 at such sizes. With the key-splitting kernels such a
// chunk took 644 us. Converting a tile during the second product instead of the first made no difference. 500 rows of 24
// heads, 8 K/V heads of 96 dims, 4000 positions, with a join: 50 us, with shares of equal work, which need two rounds of
// workgroups, 68, unsplit 101.
#include "kv_join.hpp"

namespace mtk {

constexpr int kPfKeys = 64;
constexpr int kPfRows = 128;

__device__ __forceinline__ int pf_key_order(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

template <int DT, int FMT, int DP>
__device__ __forceinline__ void kv_prefill(const mtk_kv_prefill_kargs &args) {
  const mtk_kv_attn_kargs &a = args.rows;
  constexpr int kRowB = DP * 2, kTile = kPfKeys * kRowB;
  constexpr int kKs = DP / 16, kDb = DP / 32;
  constexpr int kEl = DP == 64 ? 16 : 32;                 // dims of a thread's item
  constexpr int kIpr = DP / kEl;                          // items per key
  constexpr int kIt = kPfKeys * kIpr / 256;               // items of K (and of V) per thread and tile
  constexpr int kCh = kEl / 8;                            // 16-byte chunks per item
  constexpr int kWords = kCh * kWords8<FMT>;
  constexpr int kKeysPerWave = 64 / kIpr;                 // keys of one item index of a wavefront
  __shared__ __attribute__((aligned(1024))) char smem[4 * kTile];  // K slots 0, 1, V slots 0, 1
  // [K, V][tile & 3][wavefront][item]: lanes with a NaN block (K's are read after the tile's slot is written again)
  __shared__ uint64_t sm_bad[2][4][4][kIt];
  __shared__ int sm_nan;                                  // there was one
  __shared__ int sm_line[4][kLineWords];

  const int wg = blockIdx.x, others = (int)gridDim.x - args.joins;
  if (wg >= others) {
    kv_join<DT, false>(args.join, wg - others, args.joins, sm_line);
    return;
  }

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, col = lane & 31, G = a.G;
  if (tid == 0) sm_nan = 0;
  for (int i = tid; i < 2 * 4 * 4 * kIt; i += 256) (&sm_bad[0][0][0][0])[i] = 0;

  KvLine<kPfRows, 0> line(a, lane, sm_line[wave]);
  line.lay();
  const int64_t line_from = (int64_t)wg * line.cut.each;  // past the line's end, which 32 bits hold, for workgroups of no share
  if (line_from > INT32_MAX - line.cut.each) return;
  KvSegment seg = line.at((int)line_from, (int)line_from + line.cut.each);
  if (seg.b < 0) return;
  // As they are in every lane: else what follows from them fills vector registers, and the loads' descriptors need loops
  // (2048 rows at 8192 positions: 285 us, without 308).
  seg.seq.keys = __builtin_amdgcn_readfirstlane(seg.seq.keys);
  seg.seq.bad = __builtin_amdgcn_readfirstlane(seg.seq.bad);
  const kv_seq seq = seg.seq;
  const int rows = min(seq.rows, a.S_q) * G;
  const int r = seg.rb * kPfRows + wave * 32 + col, qi = kv_div(r, G), h = seg.hk * G + r - qi * G;
  const bool live = r < rows;

  // ---- keys: those that the workgroup's rows see, this segment's, and the last one of each row
  const int r_last = min(seg.rb * kPfRows + kPfRows, rows) - 1;
  const int64_t p_last = a.causal ? seq.pos0 + kv_div(r_last, G) : (int64_t)seq.keys - 1;
  const int n_keys = (int)max((int64_t)0, min((int64_t)seq.keys, p_last + 1));
  const int key_from = seg.from << a.step_shift, key_end = min(n_keys, seg.to << a.step_shift);
  const int n_tiles = key_end > key_from ? (key_end - key_from + kPfKeys - 1) / kPfKeys : 0;
  const int64_t pos = a.causal ? seq.pos0 + qi : (int64_t)seq.keys - 1;
  const int lim = live && pos >= 0 ? (int)min(pos, (int64_t)seq.keys - 1) : -1;
  // keys that every row of this wavefront sees (its first row the fewest)
  const int64_t w_first = a.causal ? seq.pos0 + kv_div(seg.rb * kPfRows + wave * 32, G) : (int64_t)seq.keys - 1;
  const int all_see = (int)max((int64_t)0, min((int64_t)min(seq.keys, key_end), w_first + 1));

  // ---- Q, k-steps of 16 dims; dims past D are zero
  u32x4 qf[kKs];
  {
    const uint16_t *q = (const uint16_t *)a.Q + (size_t)(seq.first + qi) * a.ld_q + (size_t)h * a.D;
#pragma unroll
    for (int ds = 0; ds < kKs; ++ds) {
      qf[ds] = u32x4{0u, 0u, 0u, 0u};
      if (live && 16 * ds + 8 * g < a.D) qf[ds] = *(const u32x4 *)(q + 16 * ds + 8 * g);
    }
  }

  // ---- staging
  const uint32_t row_b = (uint32_t)kv_row_bytes(FMT, a.blocks);
  const uint64_t region = kv_region_bytes(FMT, a.blocks, a.page_shift), page_b = region * (uint64_t)a.H_kv;
  const int page_mask = (1 << a.page_shift) - 1;
  const uint32_t k_scales = (2 * row_b) << a.page_shift, v_codes = row_b << a.page_shift;
  const uint32_t v_scales = k_scales + ((uint32_t)a.blocks << a.page_shift);
  const char *head = (const char *)a.cache + (uint64_t)(uint32_t)seg.hk * region;
  const int32_t *table = a.table + (size_t)(uint32_t)seg.b * (uint32_t)a.max_pages;
  const uint32_t pages = seq.bad ? 0u : (uint32_t)a.n_pages;
  const int last_block = (max(n_keys, 1) - 1) & ~15;
  constexpr int kWindow = 56;
  int e0 = key_from >> a.page_shift;
  int window = table[min(e0 + lane, a.max_pages - 1)], next_window = table[min(e0 + kWindow + lane, a.max_pages - 1)];

  // This thread's items: key `k_row` (K) or `v_row` (V) of each, block `blk`, chunks from `ch` on. V's keys are dealt
  // out so that the 4 keys of 16 lanes differ in bits 2 and 3, which its LDS swizzle uses.
  const int ib = tid % kIpr, ch = ib * kCh;
  const int blk = min(DP == 64 ? ib >> 1 : ib, a.blocks - 1);  // past the head's last block: that one, Q is zero there
  auto v_of = [](int k) { return (k & ~15) | ((k & 3) << 2) | ((k >> 2) & 3); };
  constexpr uint32_t kHalf = FMT == KV_FP4 ? 8 : 16;
  const uint32_t code_in = blk * 2 * kHalf + (DP == 64 ? (ib & 1) * kHalf : 0u);
  const int k_row = tid / kIpr, v_row = v_of(k_row);  // item q: + (256 / kIpr) q
  auto kswz = [](int row) { return DP >= 128 ? (row & 15) : ((row >> 1) & 7); };
  auto vswz = [](int row) {
    return DP >= 128 ? 4 * (row & 3) | ((row >> 2) & 3) : 4 * ((row >> 1) & 1) | ((row >> 2) & 3);
  };
  struct Raw {
    uint32_t w[kIt][kWords], s[kIt];
    uint32_t bad = 0;  // items whose page is not one
  };
  // Tile t's items of K (V: which 1); past the last tile: any.
  auto fetch = [&](Raw &x, int which, int t) {
    x.bad = 0;
    const int key0 = key_from + t * kPfKeys;
#pragma unroll
    for (int q = 0; q < kIt; ++q) {
      const int row = (which ? v_row : k_row) + 256 / kIpr * q;
      const int key = min(key0 + (256 / kIpr * q + kKeysPerWave * wave) / 16 * 16, last_block);
      uint32_t page = (uint32_t)__builtin_amdgcn_readlane(window, (key >> a.page_shift) - e0);
      if (page >= pages) {
        x.bad |= 1u << q;
        page = 0;
      }
      const rsrc_t rs = make_rsrc(head + (uint64_t)page * page_b, (uint32_t)region);
      const uint32_t at = (uint32_t)(key & page_mask) + (uint32_t)(row & 15);
      x.s[q] = __builtin_amdgcn_raw_buffer_load_b8(rs, at * (uint32_t)a.blocks + blk, which ? v_scales : k_scales, 0);
      const uint32_t off = at * row_b + code_in;
      if constexpr (kWords == 2) {
        const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(rs, off, which ? v_codes : 0u, 0);
        x.w[q][0] = y[0], x.w[q][1] = y[1];
      } else {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
          const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16 * i, which ? v_codes : 0u, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) x.w[q][4 * i + e] = y[e];
        }
      }
    }
  };
  // The table's windows move on before tile t is fetched (K comes first).
  auto advance = [&](int t) {
    const int key = min(key_from + t * kPfKeys + kPfKeys - 16, last_block);
    if ((key >> a.page_shift) - e0 >= 64) {
      e0 += kWindow;
      window = next_window;
      next_window = table[min(e0 + kWindow + lane, a.max_pages - 1)];
    }
  };
  bool wrote = false;  // this wavefront has written masks: from then on it writes all of them
  auto put = [&](Raw &x, int which, int slot, int t) {
    char *dst = smem + (2 * which + slot) * kTile;
    const bool tail = key_from + (t + 1) * kPfKeys > n_keys;
#pragma unroll
    for (int q = 0; q < kIt; ++q) {
      const int row = (which ? v_row : k_row) + 256 / kIpr * q;
      if (tail || wrote || x.bad || __any(x.s[q] == kNanScale)) {
        const bool past = key_from + t * kPfKeys + row >= n_keys;  // a page's unused rows may hold anything
        const bool nan = !past && (((x.bad >> q) & 1) || x.s[q] == kNanScale);
        const uint64_t nans = __ballot(nan);
        wrote = wrote || nans != 0;
        if (wrote && lane == 0) {
          sm_bad[which][t & 3][wave][q] = nans;
          sm_nan = 1;
        }
        if (nan || past) {
          x.s[q] = 127;
#pragma unroll
          for (int i = 0; i < kWords; ++i) x.w[q][i] = 0;
        }
      }
      const float scale = scale_of(x.s[q]);
#pragma unroll
      for (int f = 0; f < kCh; ++f)
        *(u32x4 *)(dst + row * kRowB + (((ch + f) ^ (which ? vswz(row) : kswz(row))) << 4)) =
            values8<DT, FMT>(x.w[q] + f * kWords8<FMT>, scale);
    }
  };
  // Keys of tile t with a NaN block (of index `only`, or any), as a bit mask. Rare.
  auto bad_keys = [&](int which, int t, int only) {
    uint64_t m = 0;
#pragma unroll 1
    for (int k = 0; k < kPfKeys; ++k) {
      const int row = which ? v_of(k) : k;  // v_of is its own inverse
      const uint64_t lanes = sm_bad[which][t & 3][(row % (256 / kIpr)) / kKeysPerWave][row / (256 / kIpr)];
      const uint32_t items = (uint32_t)(lanes >> (row % kKeysPerWave * kIpr)) & ((1u << kIpr) - 1);
      if (only < 0 ? items != 0 : ((items >> (DP == 64 ? 2 * only : only)) & 1)) m |= 1ull << k;
    }
    return m;
  };

  // ---- fragment reads
  const int krow = pf_key_order(col);
  uint32_t kq[kKs];
#pragma unroll
  for (int ds = 0; ds < kKs; ++ds) kq[ds] = (uint32_t)(krow * kRowB + (((2 * ds + g) ^ kswz(krow)) << 4));
  // V^T: lane (vh = lane / 16, vs = lane % 16) reads rows 16 js + 8 (vh / 2) + 4 e + vs / 4 at dims 32 db + 16 (vh & 1)
  // + 4 (vs & 3): the swizzle of rows 4 on differs in chunk bit 0
  const int vs = lane & 15, vh = lane >> 4;
  const int tr_row = 8 * (vh >> 1) + (vs >> 2);
  const uint32_t vq = lds_addr(smem) + (uint32_t)(2 * kTile + tr_row * kRowB + (((2 * (vh & 1) + ((vs & 3) >> 1)) ^ vswz(tr_row)) << 4) + 8 * (vs & 1));
  auto vread = [&](u32x4 (&dst)[4], uint32_t base, int db) {
    // chunk 4 db + ..: its bits are flipped in the address (DP 64: db 1's chunk bit 2 too)
    const uint32_t v0 = base ^ (uint32_t)(db << 6), v1 = v0 ^ 16u;
    static_for<0, 4>([&](auto jc) {
      constexpr int JS = decltype(jc)::value;
      const u32x2 w0 = ds_read_tr16_at<16 * kRowB * JS>(v0);
      const u32x2 w1 = ds_read_tr16_at<16 * kRowB * JS + 4 * kRowB>(v1);
      dst[JS] = u32x4{w0.x, w0.y, w1.x, w1.y};
    });
  };

  float m_off = first_offset(lim >= 0), l_run = 0.0f;
  f32x16 o[kDb];
#pragma unroll
  for (int i = 0; i < kDb; ++i) o[i] = f32x16{};
  const float c = a.scale_log2;
  constexpr int kEvery = kKs > 8 ? kKs / 8 : 1;
  constexpr int kPps = kKs >= 8 ? 1 : 8 / kKs;

  __syncthreads();  // sm_nan
  if (n_tiles > 0) {
    Raw rk, rv;
    advance(0);
    fetch(rk, 0, 0);
    fetch(rv, 1, 0);
    put(rk, 0, 0, 0);
    put(rv, 1, 0, 0);
    advance(1);
    fetch(rk, 0, 1);
    fetch(rv, 1, 1);
    __syncthreads();
    f32x16 s0 = f32x16{}, s1 = f32x16{};
#pragma unroll
    for (int ds = 0; ds < kKs; ++ds) {
      s0 = mfma32x32x16<DT>(*(const u32x4 *)(smem + kq[ds]), qf[ds], s0);
      s1 = mfma32x32x16<DT>(*(const u32x4 *)(smem + kq[ds] + 32 * kRowB), qf[ds], s1);
    }
    put(rk, 0, 1, 1);
    advance(2);
    fetch(rk, 0, 2);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = vmax3(mx, s0[i], s1[i]);

#pragma unroll 1
    for (int t = 0; t < n_tiles; ++t) {
      __syncthreads();  // K(t + 1) and V(t) are in LDS; K slot t & 1 and V slot (t + 1) & 1 are free
      const uint32_t ks = (uint32_t)(((t + 1) & 1) * kTile);
      const uint32_t vt = vq + (uint32_t)((t & 1) * kTile);
      const bool rare = sm_nan != 0;

      const int j0 = key_from + t * kPfKeys;
      if (rare) {
        const uint64_t bad = bad_keys(0, t, -1) >> (8 * g);
        const uint32_t lo = (uint32_t)bad, hi = (uint32_t)(bad >> 32);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t bit = 1u << (i < 8 ? i : i + 8);
          s0[i] = lo & bit ? __builtin_nanf("") : s0[i];
          s1[i] = hi & bit ? __builtin_nanf("") : s1[i];
        }
      }
      if (j0 + kPfKeys > all_see || rare) {
        const int last = min(lim, key_end - 1) - j0 - 8 * g;  // in the order of a lane's keys
        mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = i < 8 ? i : i + 8;
          s0[i] = k <= last ? s0[i] : -INFINITY;
          s1[i] = k + 32 <= last ? s1[i] : -INFINITY;
          mx = vmax3(mx, s0[i], s1[i]);
        }
      }
      mx = half_max(mx);
      const float m_tile = mx * c;
      float alpha = 1.0f;
      if (m_tile - m_off > kKvLift<DT> + kKvSlack) {  // a difference: exact where scores are far from zero
        alpha = __builtin_amdgcn_exp2f(m_off - (m_tile - kKvLift<DT>));
        m_off = m_tile - kKvLift<DT>;
      }
      const float moff = m_off == -INFINITY ? 0.0f : m_off;
      l_run *= alpha;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int i = 0; i < kDb; ++i) o[i] *= alpha;
      }
      put(rk, 0, t & 1, t + 2);
      put(rv, 1, (t + 1) & 1, t + 1);
      advance(t + 3);
      fetch(rk, 0, t + 3);
      fetch(rv, 1, t + 2);

      // phase A: S(t + 1) with exp / sum / pack of tile t
      __builtin_amdgcn_s_setprio(1);
      f32x16 n0 = f32x16{}, n1 = f32x16{};
      u32x4 pf[4];
      float psum = 0.0f;
      static_for<0, kKs>([&](auto dc) {
        constexpr int ds = decltype(dc)::value;
        n0 = mfma32x32x16<DT>(*(const u32x4 *)(smem + kq[ds] + ks), qf[ds], n0);
        n1 = mfma32x32x16<DT>(*(const u32x4 *)(smem + kq[ds] + ks + 32 * kRowB), qf[ds], n1);
        if constexpr ((ds + 1) % kEvery == 0) {
#pragma unroll
          for (int pp = 0; pp < kPps; ++pp) {
            const int i = 2 * ((ds / kEvery) * kPps + pp);
            const float p00 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[i], c, -moff));
            const float p01 = __builtin_amdgcn_exp2f(__builtin_fmaf(s0[i + 1], c, -moff));
            const float p10 = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[i], c, -moff));
            const float p11 = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[i + 1], c, -moff));
            psum += (p00 + p01) + (p10 + p11);
            pf[i >> 3][(i & 7) >> 1] = pack2<DT>(p00, p01);
            pf[2 + (i >> 3)][(i & 7) >> 1] = pack2<DT>(p10, p11);
          }
        }
      });
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      l_run += psum;

      // phase B: O^T += V^T(t) P^T(t) with the maxima of S(t + 1)
      constexpr int kMaxPer = kDb >= 4 ? 4 : 16 / kDb;
      u32x4 vf[2][4];
      vread(vf[0], vt, 0);
      float mn = -INFINITY;
#pragma unroll
      for (int db = 0; db < kDb; ++db) {
        const int cb = db & 1, nb = cb ^ 1;
        lgkm_wait0(vf[cb]);
        if (db + 1 < kDb) vread(vf[nb], vt, db + 1);
#pragma unroll
        for (int js = 0; js < 4; ++js) o[db] = mfma32x32x16<DT>(vf[cb][js], pf[js], o[db]);
        if (db * kMaxPer < 16) {
#pragma unroll
          for (int i = db * kMaxPer; i < db * kMaxPer + kMaxPer; ++i) mn = vmax3(mn, n0[i], n1[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (rare) {  // the dims of a NaN block, for the rows that see the key
        const int seen = lim - j0 + 1;
        const uint64_t vis = seen >= 64 ? ~0ull : seen <= 0 ? 0ull : (1ull << seen) - 1;
#pragma unroll
        for (int db = 0; db < kDb; ++db)
          if (bad_keys(1, t, db) & vis) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] = __builtin_nanf("");
          }
      }
      s0 = n0;
      s1 = n1;
      mx = mn;
    }
  }

  // ---- O[row][h][d] = O^T[d][row] / l, or this workgroup's part
  const float l_tot = half_sum(l_run);
  if (!live) return;
  if (seg.from == 0 && seg.to == seg.steps) {
    const float inv = inverse_of(l_tot, m_off);
    uint16_t *O = (uint16_t *)a.O + ((size_t)(seq.first + qi) * a.H + h) * a.D;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 32 * db + 8 * q + 4 * g;
        if (d < a.D)
          *(u32x2 *)(O + d) = u32x2{pack2<DT>(o[db][4 * q] * inv, o[db][4 * q + 1] * inv),
                                    pack2<DT>(o[db][4 * q + 2] * inv, o[db][4 * q + 3] * inv)};
      }
    if (g == 0 && a.lse)
      a.lse[(size_t)(seq.first + qi) * a.H + h] =
          l_tot == 0.0f ? -INFINITY : (m_off == -INFINITY ? l_tot : m_off + __builtin_amdgcn_logf(l_tot)) * 0.6931471805599453f;
  } else if (wg < a.places) {
    const size_t at = (size_t)wg * kPfRows + wave * 32 + col;
    float *x = a.part + at * a.part_ld;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * db < a.part_ld)
          *(f32x4 *)(x + 32 * db + 8 * q + 4 * g) = f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]};
    if (g == 0) *(f32x2 *)(a.part_ml + 2 * at) = f32x2{m_off, l_tot};
  }
}

}  // namespace mtk

using namespace mtk;

// mtk_kv_prefill_<format>_d<padded head dimension>_<type>: two workgroups per CU, or one (D above 128)
#define MTK_KV_PREFILL(NAME, DT, FMT, DP, EU)                                                       \
  extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(EU, EU)))   \
  NAME(const mtk_kv_prefill_kargs a) { kv_prefill<DT, FMT, DP>(a); }
#define MTK_KV_PREFILL_DP(DP, EU)                                          \
  MTK_KV_PREFILL(mtk_kv_prefill_fp4_d##DP##_f16, DT_F16, KV_FP4, DP, EU)   \
  MTK_KV_PREFILL(mtk_kv_prefill_fp4_d##DP##_bf16, DT_BF16, KV_FP4, DP, EU) \
  MTK_KV_PREFILL(mtk_kv_prefill_fp8_d##DP##_f16, DT_F16, KV_FP8, DP, EU)   \
  MTK_KV_PREFILL(mtk_kv_prefill_fp8_d##DP##_bf16, DT_BF16, KV_FP8, DP, EU)
MTK_KV_PREFILL_DP(64, 2)
MTK_KV_PREFILL_DP(128, 2)
MTK_KV_PREFILL_DP(256, 1)
