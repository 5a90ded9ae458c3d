// Plans of the paged key/value cache in few bits (include/mtk.h, kv_cache.h): checks, kernel choice and argument
// blocks. Part of runtime.cpp's translation unit, inside its unnamed namespace.

constexpr int kKvMaxPositions = 1 << 30;  // of a table row

bool is_kv(const mtk_plan *p) { return p->kind == PLAN_KV_WRITE || p->kind == PLAN_KV_READ || p->kind == PLAN_KV_ATTN; }

int kv_blocks_of(const mtk_kv_desc &d) { return (d.D + 31) / 32; }
int kv_shift_of(const mtk_kv_desc &d) { return __builtin_ctz((unsigned)d.page_size); }
uint64_t kv_cache_size(const mtk_kv_desc &d) {
  return (uint64_t)d.n_pages * (uint64_t)d.H_kv * kv_region_bytes(d.format, kv_blocks_of(d), kv_shift_of(d));
}

int check_kv_geometry(const mtk_kv_desc &d) {
  if (d.H_kv <= 0 || d.n_pages <= 0) return fail(MTK_ERR_INVALID, "H_kv and n_pages must be positive (got %d, %d)", d.H_kv, d.n_pages);
  if (d.D <= 0 || d.D > 256 || d.D % 8 != 0)
    return fail(MTK_ERR_UNSUPPORTED, "head dimension must be a multiple of 8 up to 256 (got %d)", d.D);
  if (d.page_size < 16 || d.page_size > 1024 || (d.page_size & (d.page_size - 1)) != 0)
    return fail(MTK_ERR_INVALID, "page_size must be a power of two from 16 to 1024 (got %d)", d.page_size);
  if (d.format != MTK_KV_FP4 && d.format != MTK_KV_FP8) return fail(MTK_ERR_INVALID, "format must be MTK_KV_FP4 or MTK_KV_FP8");
  if (d.H_kv > (1 << 20)) return fail(MTK_ERR_UNSUPPORTED, "H_kv above %d is not supported", 1 << 20);
  if ((double)d.n_pages * d.H_kv * (double)kv_region_bytes(d.format, kv_blocks_of(d), kv_shift_of(d)) > 9e18)
    return fail(MTK_ERR_UNSUPPORTED, "a cache of this size cannot be addressed");
  return MTK_OK;
}

// What the three plans have in common.
int check_kv_batch(const mtk_kv_desc &d) {
  const int s = check_kv_geometry(d);
  if (s != MTK_OK) return s;
  if (d.B <= 0 || d.T <= 0 || d.max_pages <= 0)
    return fail(MTK_ERR_INVALID, "B, T and max_pages must be positive (got %d, %d, %d)", d.B, d.T, d.max_pages);
  if ((long long)d.max_pages * d.page_size > kKvMaxPositions)
    return fail(MTK_ERR_UNSUPPORTED, "a table row of more than 2^30 positions is not supported");
  if (d.dtype != MTK_F16 && d.dtype != MTK_BF16) return fail(MTK_ERR_INVALID, "dtype must be MTK_F16 or MTK_BF16");
  return MTK_OK;
}

int kv_ld(int ld, int width, const char *name, int64_t *out) {
  *out = ld ? ld : width;
  if (ld != 0 && (ld < width || ld % 8 != 0))
    return fail(MTK_ERR_INVALID, "%s must be 0 or a multiple of 8 of at least %d (got %d)", name, width, ld);
  return MTK_OK;
}

std::string kv_suffix(const mtk_kv_desc &d) { return d.dtype == MTK_F16 ? "f16" : "bf16"; }
const char *kv_format(const mtk_kv_desc &d) { return d.format == MTK_KV_FP4 ? "fp4" : "fp8"; }

int finish_kv(mtk_plan *p, mtk_plan **out) {
  const int s = resolve(p);
  if (s != MTK_OK) {
    delete p;
    return s;
  }
  *out = p;
  return MTK_OK;
}

int plan_kv_move(mtk_ctx *ctx, const mtk_kv_desc *d_in, PlanKind kind, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  const mtk_kv_desc d = *d_in;
  int s = check_kv_batch(d);
  if (s != MTK_OK) return s;
  mtk_kv_move_kargs a{};
  if ((s = kv_ld(d.ld_k, d.H_kv * d.D, "ld_k", &a.ld_k)) != MTK_OK || (s = kv_ld(d.ld_v, d.H_kv * d.D, "ld_v", &a.ld_v)) != MTK_OK) return s;
  a.B = d.B;
  a.T = d.T;
  a.H_kv = d.H_kv;
  a.D = d.D;
  a.blocks = kv_blocks_of(d);
  a.page_shift = kv_shift_of(d);
  a.n_pages = d.n_pages;
  a.max_pages = d.max_pages;
  const long long items = 8LL * d.H_kv * a.blocks;  // of 16 bytes of K or V, per row
  // Up to KV_MOVE_ROWS rows per wavefront, whose places it looks up once and whose lines in the cache it fills itself; fewer where
  // that would leave less than 8 wavefronts per CU. 64 items of each.
  const int cus = ctx ? ctx->prop.multiProcessorCount : 256;
  a.parts = (int)((items + 63) / 64);
  a.rows_per_wave = 1;
  while (a.rows_per_wave < KV_MOVE_ROWS && (d.T + 2LL * a.rows_per_wave - 1) / (2 * a.rows_per_wave) * a.parts >= 8LL * cus) a.rows_per_wave *= 2;
  const long long groups = ((long long)d.T + a.rows_per_wave - 1) / a.rows_per_wave;
  a.mul_blocks = a.blocks == 1 ? 0u : (uint32_t)((0x100000000ull + a.blocks - 1) / a.blocks);
  const long long waves = a.parts * groups;
  if ((waves + 3) / 4 > INT32_MAX / 256) return fail(MTK_ERR_UNSUPPORTED, "T of %d is not supported", d.T);
  mtk_plan *p = new mtk_plan();
  p->ctx = ctx;
  p->kind = kind;
  p->kv = d;
  Launch g;
  g.name = std::string(kind == PLAN_KV_WRITE ? "mtk_kv_write_" : "mtk_kv_read_") + kv_format(d) + "_" + kv_suffix(d);
  g.grid = (unsigned)((waves + 3) / 4);
  set_args(g, a);
  p->launches.push_back(g);
  p->bytes = (double)d.T * d.H_kv * (4.0 * d.D + 2.0 * (kv_row_bytes(d.format, a.blocks) + a.blocks)) + 4.0 * (2.0 * d.B + 1);
  char desc[256];
  snprintf(desc, sizeof desc, "kv %s %s %s B=%d T=%d H_kv=%d D=%d pages=%dx%d max_pages=%d waves/row=%d rows/wave=%d grid=%u",
           kind == PLAN_KV_WRITE ? "write" : "read", kv_format(d), kv_suffix(d).c_str(), d.B, d.T, d.H_kv, d.D, d.n_pages,
           d.page_size, d.max_pages, a.parts, a.rows_per_wave, g.grid);
  p->description = desc;
  return finish_kv(p, out);
}

// Of the attention kernels (kv_attention.hip): keys per tile, wavefronts per workgroup, workgroups per CU as their registers
// and LDS allow. Measured for 32 rows of (row, query head) pairs, fp4, 128 dims (8 x 3000 to 8000 positions, the first
// kernel): 32 keys, 8 wavefronts, 1 workgroup 22.3 us; 4 and 2 22.8; 64 keys, 8 and 1 23.7; 64 keys, 4 and 2 24.1.
struct KvShape {
  int tile, waves, per_cu;
  int step() const { return tile * waves; }
};
KvShape kv_kernel_shape(int fmt, int dp, int nr) {
  const bool fp4 = fmt == MTK_KV_FP4;
  if (nr == 4) return {32, 4, dp == 64 ? 2 : 1};
  if (dp == 64) return nr == 1 ? KvShape{64, 4, fp4 ? 4 : 3} : KvShape{64, 8, 1};
  if (dp == 128) return nr == 1 ? KvShape{32, 4, fp4 ? 4 : 3} : KvShape{32, 8, 1};
  return nr == 1 ? KvShape{32, 8, 1} : KvShape{32, 4, 1};
}

int plan_kv_attn(mtk_ctx *ctx, const mtk_kv_desc *d_in, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  mtk_kv_desc d = *d_in;
  int s = check_kv_batch(d);
  if (s != MTK_OK) return s;
  if (d.H <= 0 || d.H % d.H_kv != 0) return fail(MTK_ERR_INVALID, "H must be a positive multiple of H_kv (got H=%d, H_kv=%d)", d.H, d.H_kv);
  if (d.S_q == 0) d.S_q = d.T;
  if (d.S_q < 0 || d.S_q > d.T) return fail(MTK_ERR_INVALID, "S_q must be 0 to T (got %d, T=%d)", d.S_q, d.T);
  if ((long long)d.S_q * (d.H / d.H_kv) > INT32_MAX / 2)
    return fail(MTK_ERR_UNSUPPORTED, "S_q x H / H_kv of %lld is not supported", (long long)d.S_q * (d.H / d.H_kv));
  if ((long long)d.H * d.D > INT32_MAX || (long long)d.T * d.H > INT32_MAX / 64)
    return fail(MTK_ERR_UNSUPPORTED, "T x H of more than 2^25 rows, or rows of more than 2^31 elements, are not supported");
  mtk_kv_attn_kargs a{};
  if ((s = kv_ld(d.ld_q, d.H * d.D, "ld_q", &a.ld_q)) != MTK_OK) return s;
  const int G = d.H / d.H_kv, cus = ctx ? ctx->prop.multiProcessorCount : 256;
  const int dp = d.D <= 64 ? 64 : d.D <= 128 ? 128 : 256;
  a.B = d.B;
  a.T = d.T;
  a.S_q = d.S_q;
  a.H = d.H;
  a.H_kv = d.H_kv;
  a.G = G;
  a.D = d.D;
  a.blocks = kv_blocks_of(d);
  a.page_shift = kv_shift_of(d);
  a.n_pages = d.n_pages;
  a.max_pages = d.max_pages;
  a.causal = d.causal ? 1 : 0;
  a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)d.D));
  a.part_ld = a.blocks * 32;
  const long long positions = (long long)d.max_pages * d.page_size;
  const long long pairs = (long long)d.S_q * G;  // (row, query head) pairs of a sequence and K/V head, at most
  // Sequences of up to 64 pairs: kernels whose wavefronts split the keys. Others: kernels whose wavefronts split the
  // rows, and the former for the sequences that have one new row (or few) all the same.
  const int most = dp == 256 ? 32 : 64;
  const int few = pairs <= most ? (int)pairs : G <= most ? G : 0;
  std::vector<Launch> launches;
  size_t workspace = 0;
  std::string how;
  char name[96];
  // Partial sums of a launch with `grid` workgroups. Run-time pointers: offsets in the workspace until then.
  auto partial_sums = [&](mtk_kv_attn_kargs &k, long long grid) {
    k.places = (int)grid;
    const size_t held = (size_t)grid * (k.by_pair ? 1 : 2) << k.rows_shift;
    const size_t part = workspace, ml = part + held * k.part_ld * sizeof(float);
    workspace = ml + held * 2 * sizeof(float);
    k.part = (float *)part;
    k.part_ml = (float *)ml;
  };
  // Workgroups that join them with the lanes over the heads, or in a launch of its own over the parts of each (row, head):
  // where a pair has more than 8 parts and there are few (row, head)s to fill the device with. 1 x 131071 positions, 8 K/V heads:
  // both kernels 35.5 us, over the heads 49.6; 4 x 8000: 17.6 and 20.1; but 4 x 2000 with 16 rows of 16 heads: 23.0 and 20.7,
  // 16 x 8000: 35.9 and 34.6.
  auto joins = [&](const mtk_kv_attn_kargs &k, bool parts, int most_wgs) {
    const long long mine = k.by_pair ? d.T : std::min<long long>(d.T, (long long)d.B * std::max(1, k.rows_most / G));
    const int heads = parts ? 1 : 1024 / k.part_ld;
    return (int)std::min<long long>(mine * ((d.H + heads - 1) / heads), most_wgs);
  };
  auto add = [&](const std::string &kernel, long long grid, int block, const auto &args) {
    Launch g;
    g.name = kernel;
    g.grid = (unsigned)grid;
    g.block = (unsigned)block;
    set_args(g, args);
    launches.push_back(g);
  };
  // At most 4 workgroups per CU, which are there at once: 2 x 500 rows of 32 heads in two parts 16.8 us, 8 per CU 19.6, 2 17.9.
  auto add_join = [&](const mtk_kv_attn_kargs &k, bool parts) {
    add(std::string(parts ? "mtk_kv_join_parts_" : "mtk_kv_join_rows_") + kv_suffix(d), joins(k, parts, 4 * cus), 256, k);
  };
  auto tell = [&](int rows, long long grid, bool split) {
    char text[96];
    snprintf(text, sizeof text, " rows/wg=%d grid=%lld%s", rows, grid, split ? " keys split" : "");
    how += text;
  };
  auto too_large = [&](long long blocks, long long steps) {
    return blocks >= (1 << 23) || blocks * steps > INT32_MAX
               ? fail(MTK_ERR_UNSUPPORTED, "a batch of %lld row blocks over %lld positions is not supported", blocks, positions)
               : MTK_OK;
  };
  mtk_kv_attn_kargs k = a;  // of the sequences with few rows
  if (few) {
    const int nr = few <= 16 ? 1 : few <= 32 || dp == 256 ? 2 : 4, rows = 16 * nr;
    // Few pairs of short sequences: one workgroup of 16 wavefronts each, no second kernel. 1000 positions, 8 pairs: 9.0 us
    // against 12.0 with the keys split; 32 x 4000 (256 pairs): 26.8 and 32.5; but 4 x 4000 (32 pairs): 19.6 and 14.3. Longer
    // tables would gain too where pairs fill the device and are equally long (32 x 8000: 53.6 and 62.3), not where one is long.
    // The lengths lie on the device, so that the table's capacity stands for them here: short sequences behind a long table
    // take the split kernels.
    const long long blocks = (long long)d.B * d.H_kv;
    const bool wide = nr == 1 && dp <= 128 && blocks <= cus && positions <= (2 * blocks >= cus ? 4096 : 2048);
    const KvShape shape = wide ? KvShape{32, 16, 1} : kv_kernel_shape(d.format, dp, nr);
    k.rows_above = 0;
    k.rows_most = rows;
    k.rows_shift = __builtin_ctz((unsigned)rows);
    k.step_shift = __builtin_ctz((unsigned)shape.step());
    k.units = cus * shape.per_cu;
    k.least = 2;  // 1 x 16000: 14.7 us, least 1: 16.9; 4 x 2000 with 16 rows: 23.0, least 4: 25.1
    const long long steps = (positions + shape.step() - 1) / shape.step();
    if ((s = too_large(blocks, 2 * (steps + k.least))) != MTK_OK) return s;
    // 64 x 1000: whole pairs 16.3 us, split 22.1; 64 x 2000 (512 pairs): 28.3 and 32.5; 8 x 4000 with 16 rows: 80 and 34
    k.whole = wide || positions <= (blocks >= 2 * cus ? 2048 : 1024) ? 1 : 0;
    snprintf(name, sizeof name, "mtk_kv_attend_%s_d%d_r%d_%s%s", kv_format(d), dp, nr, wide ? "w16_" : "", kv_suffix(d).c_str());
    const long long grid = k.whole ? blocks : k.units;
    if (!k.whole) partial_sums(k, grid);
    add(name, grid, 64 * shape.waves, k);
    tell(rows, grid, !k.whole);
    if (!k.whole && pairs <= most) add_join(k, blocks * 8 < grid && (long long)joins(k, true, INT32_MAX) < 2LL * cus);
  }
  if (pairs > most) {
    const int rows = 128;
    mtk_kv_prefill_kargs both{};
    mtk_kv_attn_kargs &r = both.rows;
    r = a;
    r.rows_above = few ? k.rows_most : 0;
    r.rows_most = INT32_MAX;
    r.by_pair = 1;
    r.units = cus * (dp == 256 ? 1 : 2);
    const long long each = (long long)d.B * ((pairs + rows - 1) / rows) * d.H_kv;  // blocks, whatever row_start holds
    const long long blocks = kv_max_blocks(d.B, d.T, d.S_q, G, rows) * d.H_kv;
    // Fewer blocks than workgroups: the keys are split, into 4 steps (256 keys) or more, so that all workgroups are on the
    // device at once; else never. 300 rows of 8 heads of 64 dims, 1000 positions: 17.8 us, 8 steps 22.6, 2 steps 16.8;
    // 2 x 4000 positions, 100 rows, 256 dims: 47.4, 54.8 and 47.3, with shares of equal work (two rounds) 51.3, unsplit 215.
    // Decided on the device; here only whether the blocks may be so few, each sequence's last one aside.
    const bool split = std::min(blocks, (long long)d.T * G / rows * d.H_kv) < r.units && positions > 256;
    const kv_pair_steps steps = kv_steps_of_pairs(each, positions, split);
    if (steps.shift < 0 || blocks >= (1 << 23))
      return fail(MTK_ERR_UNSUPPORTED, "a batch of %lld row blocks is not supported", steps.shift < 0 ? each : blocks);
    r.least = steps.least;
    r.step_shift = steps.shift;
    r.rows_shift = __builtin_ctz((unsigned)rows);
    const long long grid = split ? std::max<long long>(r.units, blocks) : blocks;
    if (split) partial_sums(r, r.units);
    // The sums that the launch before has left are joined by this one's last workgroups, at most one per CU, beside the
    // others: 500 rows at 4000 positions and 31 tokens at 8000 106.6 us, with a launch of their own 112.8.
    if (k.places) {
      both.join = k;
      both.joins = joins(k, false, cus);
    }
    snprintf(name, sizeof name, "mtk_kv_prefill_%s_d%d_%s", kv_format(d), dp, kv_suffix(d).c_str());
    add(name, grid + both.joins, 256, both);
    tell(rows, grid, split);
    if (split) add_join(r, false);
  }
  mtk_plan *p = new mtk_plan();
  p->ctx = ctx;
  p->kind = PLAN_KV_ATTN;
  p->kv = d;
  p->launches = launches;
  p->workspace = workspace;
  const double cap = (double)positions;
  p->flops = 4.0 * d.T * d.H * d.D * cap;
  p->bytes = d.B * cap * d.H_kv * 2.0 * (kv_row_bytes(d.format, a.blocks) + a.blocks) + 4.0 * d.T * d.H * d.D +
             4.0 * (2.0 * d.B + 1 + (double)d.B * d.max_pages);
  char desc[320];
  snprintf(desc, sizeof desc, "kv attention %s %s B=%d T=%d S_q=%d H=%d H_kv=%d D=%d pages=%dx%d max_pages=%d causal=%d", kv_format(d),
           kv_suffix(d).c_str(), d.B, d.T, d.S_q, d.H, d.H_kv, d.D, d.n_pages, d.page_size, d.max_pages, a.causal);
  p->description = desc + how;
  return finish_kv(p, out);
}

// ------------------------------------------------------------------ run-time arguments

bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y ? a_bytes > y - x : b_bytes > x - y;
}

// Bytes that `rows` rows of `width` elements with `ld` between them span.
uint64_t kv_span(int rows, int64_t ld, int64_t width) { return 2 * ((uint64_t)(rows - 1) * (uint64_t)ld + (uint64_t)width); }

// Whether one of n rows of `width` elements from a on, `ld_a` apart, meets one of as many from b on: slices of one buffer lie
// between each other.
bool rows_meet(const void *a, int64_t ld_a, const void *b, int64_t ld_b, int n, int64_t width) {
  if (!overlap(a, kv_span(n, ld_a, width), b, kv_span(n, ld_b, width))) return false;
  const uint64_t x = (uintptr_t)a, y = (uintptr_t)b, bytes = 2 * (uint64_t)width, step_a = 2 * (uint64_t)ld_a, step_b = 2 * (uint64_t)ld_b;
  if (ld_a == ld_b) {  // the distances of their rows: |x - y| less so many strides
    const uint64_t apart = x < y ? y - x : x - y, rows = apart / step_a, rest = apart % step_a;
    return (rest < bytes && rows < (uint64_t)n) || (step_a - rest < bytes && rows + 1 < (uint64_t)n);
  }
  for (int i = 0, j = 0; i < n && j < n;) {
    const uint64_t s = x + (uint64_t)i * step_a, t = y + (uint64_t)j * step_b;
    if (s < t ? t - s < bytes : s - t < bytes) return true;
    s < t ? ++i : ++j;
  }
  return false;
}

int check_kv_args(const mtk_plan *p, const void *argset) {
  const mtk_kv_desc &d = p->kv;
  struct Buffer {
    const char *name;
    const void *at;
    uint64_t bytes;
  };
  Buffer in[5] = {}, out[3] = {};  // what the operator reads and writes
  const int32_t *ints[3];
  const void *cache;
  if (!argset) return fail(MTK_ERR_INVALID, "null arguments");
  if (p->kind == PLAN_KV_ATTN) {
    const mtk_kv_attn_args *t = (const mtk_kv_attn_args *)argset;
    cache = t->cache;
    ints[0] = t->row_start, ints[1] = t->kv_len, ints[2] = t->table;
    if (!t->Q || !t->O) return fail(MTK_ERR_INVALID, "Q and O must be non-null");
    if (!aligned(t->Q, 16) || !aligned(t->O, 16)) return fail(MTK_ERR_INVALID, "Q and O must be 16-byte aligned");
    if (t->lse && !aligned(t->lse, 4)) return fail(MTK_ERR_INVALID, "lse must be 4-byte aligned");
    if (p->workspace && (!t->workspace || !aligned(t->workspace, 16)))
      return fail(MTK_ERR_INVALID, "this plan needs a 16-byte aligned workspace of %zu bytes", p->workspace);
    const int64_t width = (int64_t)d.H * d.D;
    in[0] = {"Q", t->Q, kv_span(d.T, d.ld_q ? d.ld_q : width, width)};
    in[1] = {"the cache", cache, kv_cache_size(d)};
    out[0] = {"O", t->O, kv_span(d.T, width, width)};
    out[1] = {"lse", t->lse, 4ull * d.T * d.H};
    out[2] = {"the workspace", t->workspace, p->workspace};
  } else {
    const bool write = p->kind == PLAN_KV_WRITE;
    const mtk_kv_write_args *w = (const mtk_kv_write_args *)argset;
    const mtk_kv_read_args *r = (const mtk_kv_read_args *)argset;
    const void *K = write ? w->K : r->K, *V = write ? w->V : r->V;
    cache = write ? w->cache : r->cache;
    ints[0] = write ? w->row_start : r->row_start, ints[1] = write ? w->kv_len : r->kv_len, ints[2] = write ? w->table : r->table;
    if (!K || !V) return fail(MTK_ERR_INVALID, "K and V must be non-null");
    if (!aligned(K, 16) || !aligned(V, 16)) return fail(MTK_ERR_INVALID, "K and V must be 16-byte aligned");
    const int64_t width = (int64_t)d.H_kv * d.D, ld_k = d.ld_k ? d.ld_k : width, ld_v = d.ld_v ? d.ld_v : width;
    if (!write && K == V) return fail(MTK_ERR_INVALID, "K and V are the same rows");
    if (!write && rows_meet(K, ld_k, V, ld_v, d.T, width)) return fail(MTK_ERR_INVALID, "K overlaps V");
    const Buffer rows[2] = {{"K", K, kv_span(d.T, ld_k, width)}, {"V", V, kv_span(d.T, ld_v, width)}}, held = {"the cache", cache, kv_cache_size(d)};
    (write ? in : out)[0] = rows[0];
    (write ? in : out)[1] = rows[1];
    (write ? out : in)[2] = held;
  }
  if (!cache || !aligned(cache, 16)) return fail(MTK_ERR_INVALID, "the cache must be non-null and 16-byte aligned");
  for (const int32_t *x : ints)
    if (!x || !aligned(x, 4)) return fail(MTK_ERR_INVALID, "row_start, kv_len and table must be non-null and 4-byte aligned");
  const Buffer arrays[3] = {{"row_start", ints[0], 4 * ((uint64_t)d.B + 1)}, {"kv_len", ints[1], 4 * (uint64_t)d.B},
                            {"the table", ints[2], 4 * (uint64_t)d.B * (uint64_t)d.max_pages}};
  for (int i = 0; i < 3; ++i) {
    const Buffer &o = out[i];
    if (!o.at || !o.bytes) continue;
    auto meets = [&](const Buffer &x) { return x.at && overlap(o.at, o.bytes, x.at, x.bytes); };
    for (const Buffer &x : in)
      if (meets(x)) return fail(MTK_ERR_INVALID, "%s overlaps %s", p->kind == PLAN_KV_WRITE ? x.name : o.name, p->kind == PLAN_KV_WRITE ? o.name : x.name);
    for (const Buffer &x : arrays)
      if (meets(x)) return fail(MTK_ERR_INVALID, "%s overlaps %s", o.name, x.name);
    for (int k = 0; p->kind == PLAN_KV_ATTN && k < i; ++k)
      if (meets(out[k])) return fail(MTK_ERR_INVALID, "%s overlaps %s", o.name, out[k].name);
  }
  return MTK_OK;
}

// Writes the run-time pointers of a launch into `block`, a copy of its argument block.
void patch_kv(const mtk_plan *p, const Launch &l, char *block, const void *argset) {
  if (p->kind == PLAN_KV_ATTN) {
    const mtk_kv_attn_args *t = (const mtk_kv_attn_args *)argset;
    mtk_kv_attn_kargs *const all = (mtk_kv_attn_kargs *)block;  // two of them: mtk_kv_prefill_kargs
    for (int i = 0; i < (l.args.size() == sizeof(mtk_kv_prefill_kargs) ? 2 : 1); ++i) {
      mtk_kv_attn_kargs &a = all[i];
      a.Q = t->Q;
      a.cache = t->cache;
      a.row_start = t->row_start;
      a.kv_len = t->kv_len;
      a.table = t->table;
      a.O = t->O;
      a.lse = t->lse;
      a.part = (float *)((uintptr_t)a.part + (uintptr_t)t->workspace);
      a.part_ml = (float *)((uintptr_t)a.part_ml + (uintptr_t)t->workspace);
    }
    return;
  }
  mtk_kv_move_kargs &a = *(mtk_kv_move_kargs *)block;
  if (p->kind == PLAN_KV_WRITE) {
    const mtk_kv_write_args *t = (const mtk_kv_write_args *)argset;
    a.K = t->K;
    a.V = t->V;
    a.cache = t->cache;
    a.row_start = t->row_start;
    a.kv_len = t->kv_len;
    a.table = t->table;
  } else {
    const mtk_kv_read_args *t = (const mtk_kv_read_args *)argset;
    a.K = t->K;
    a.V = t->V;
    a.cache = const_cast<void *>(t->cache);
    a.row_start = t->row_start;
    a.kv_len = t->kv_len;
    a.table = t->table;
  }
}

// A run: argument blocks on the stack, nothing is allocated.
int run_kv(const mtk_plan *p, PlanKind kind, const void *argset) {
  if (!p) return fail(MTK_ERR_INVALID, "null plan");
  if (p->kind != kind)
    return fail(MTK_ERR_INVALID, "not a plan for %s",
                kind == PLAN_KV_WRITE ? "writing a cache" : kind == PLAN_KV_READ ? "reading a cache" : "attention over a cache");
  if (!p->ctx) return fail(MTK_ERR_INVALID, "plan was created without a context (dry plan)");
  const int s = check_kv_args(p, argset);
  if (s != MTK_OK) return s;
  alignas(16) char block[512];
  HIP_TRY(hipSetDevice(p->ctx->device));
  for (const Launch &l : p->launches) {
    if (l.args.size() > sizeof block) return fail(MTK_ERR_INVALID, "argument block of %s too large", l.name.c_str());
    memcpy(block, l.args.data(), l.args.size());
    patch_kv(p, l, block, argset);
    void *params[] = {block};
    const hipError_t e = hipModuleLaunchKernel(l.fn, l.grid, 1, 1, l.block, 1, 1, 0, p->ctx->stream, params, nullptr);
    if (e != hipSuccess) return fail(MTK_ERR_LAUNCH, "launch of %s failed: %s", l.name.c_str(), hipGetErrorString(e));
  }
  return MTK_OK;
}
