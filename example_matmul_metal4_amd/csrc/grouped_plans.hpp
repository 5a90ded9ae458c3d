// Plans of products grouped by expert and of rows and products in few bits (include/mtk.h, groups.h, mx.h): checks, kernel
// choice and argument blocks. Part of runtime.cpp's translation unit, inside its unnamed namespace.

constexpr int kMaxWidth = 1 << 22;  // N, K and leading dimensions: 256 rows of a tile, and 64 past an operand's end, stay in 32 bits
constexpr int kMaxGroups = 1 << 14;  // a workgroup looks through all of them, 64 at a time
constexpr int kMaxRows = 1 << 30;    // counts of rows, rounded up to blocks, stay in 32 bits

bool is_grouped(const mtk_plan *p) { return p->kind >= PLAN_GROUPED && p->kind <= PLAN_MX_GEMM; }

int check_ld(int ld, int width, const char *name, int *out) {
  *out = ld ? ld : width;
  if (ld != 0 && ld < width) return fail(MTK_ERR_INVALID, "%s must be 0 or at least %d (got %d)", name, width, ld);
  if (*out > kMaxWidth) return fail(MTK_ERR_UNSUPPORTED, "%s of more than 2^22 (%d) is not supported", name, *out);
  return MTK_OK;
}

int finish_plan(std::unique_ptr<mtk_plan> p, mtk_plan **out) {
  const int s = resolve(p.get());
  if (s == MTK_OK) *out = p.release();
  return s;
}

// No exception leaves a C entry point: making a plan allocates.
template <typename F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return fail(MTK_ERR_OOM, "out of memory");  // short enough for the error string to hold without allocating
  } catch (...) {
    return fail(MTK_ERR_INVALID, "unexpected exception");
  }
}

template <typename T>
void add_launch(mtk_plan *p, const std::string &name, long long grid, int block, const T &args) {
  Launch l;
  l.name = name;
  l.grid = (unsigned)grid;
  l.block = (unsigned)block;
  set_args(l, args);
  p->launches.push_back(l);
}

int check_grouped(const mtk_grouped_desc &d) {
  if (d.E <= 0 || d.T <= 0 || d.N <= 0 || d.K <= 0)
    return fail(MTK_ERR_INVALID, "E, T, N and K must be positive (got %d, %d, %d, %d)", d.E, d.T, d.N, d.K);
  if (d.N > kMaxWidth || d.K > kMaxWidth) return fail(MTK_ERR_UNSUPPORTED, "N and K above 2^22 are not supported (got %d, %d)", d.N, d.K);
  if (d.E > kMaxGroups) return fail(MTK_ERR_UNSUPPORTED, "E above 2^14 is not supported (got %d)", d.E);
  if (d.T > kMaxRows) return fail(MTK_ERR_UNSUPPORTED, "T above 2^30 is not supported (got %d)", d.T);
  if (d.dtype != MTK_F16 && d.dtype != MTK_BF16) return fail(MTK_ERR_INVALID, "dtype must be MTK_F16 or MTK_BF16");
  return MTK_OK;
}

// Workgroups of the tiles that expert_tiles.hpp runs: as many as are on the device at once, each with one tile after another.
long long tile_grid(int tile, int cus, long long tiles) {
  return tile <= 64 ? tiles : std::min<long long>(tiles, (tile == 128 ? 2LL : 1LL) * cus);
}

// A launch has fewer than 2^32 threads.
bool launches(long long grid, int threads) { return grid <= (long long)(UINT32_MAX / (unsigned)threads); }

// A launch that finds its tiles from row_start: workgroups for all that ascending groups can have. fits: the launch can have so many, and no
// count of tiles passes 32 bits whatever row_start holds (every group may have all rows).
struct TileCount {
  long long grid;
  bool fits;
};
TileCount count_tiles(int E, int T, int tile, int waves, long long tiles_n, int cus) {
  TileCount c;
  c.grid = tile_grid(tile, cus, group_max_blocks(E, T, tile) * tiles_n);
  c.fits = (long long)E * (((long long)T + tile - 1) / tile) * tiles_n <= INT32_MAX && launches(c.grid, 64 * waves);
  return c;
}

// Which kernel runs a product, by the time that it is expected to take, in us: `start` and the larger of
//   rounds * (round + (step + full * part) * K-tiles of a wavefront)   and   bytes * byte (us per MB),
// with 0.15 of the other. rounds: workgroups over those that are on the device at once, between that and the next whole number, at
// least 1; part: that share, at most 1 (a full device's K-tiles take longer). The groups' sizes lie on the device: of E groups,
// E (1 - exp(-T / E)) are taken to have rows, as if each row chose one of E, and each to have half a block that is not full. Fitted
// to launches of 400 forward products, 300 gradients and 350 products in few bits, each by every kernel (random sizes, T to 16384,
// N and K 64 to 14336): the kernel chosen takes 1.02, 1.04 and 1.01 times (geometric mean) the time of the fastest.
// Examples, us (tiles of 256, of 128, of 64 with 8, 4, 1 wavefronts): 256 rows over 8 groups of 14336 x 4096: 191, 163, 157, 155, 149;
// 8192 over 16 of 4096 x 4096: 292, 335, 605, 534, 518; 16 over 32 of 2048 x 2048: 29, 22, 22, 19, 39. Gradients: 8192 over 16 of 4096
// x 4096: 294, 352, 1289, 777, 593; 1000 over 24 of 1023 x 520 with the bias': -, -, 56, 36, 27.
struct TileCost {
  int tile, waves, per_cu;  // rows and columns of a tile (32: 64 columns); wavefronts and workgroups per CU
  double start, round, step, full, byte;
  double any;  // odd leading dimensions: K-tiles take longer by this share; below 0: not for these
};
constexpr TileCost kForward[] = {{256, 8, 1, 4.9, 0.0, 0.75, 1.06, 0.24, -1},
                                 {128, 4, 2, 1.1, 3.31, 0.51, 0.66, 0.17, -1},
                                 {64, 8, 1, 1.7, 1.40, 1.35, 0.87, 0.17, 0.18},
                                 {64, 4, 2, 1.7, 2.18, 0.83, 1.06, 0.17, 0.27},
                                 {64, 1, 8, 0.0, 4.38, 0.77, 1.03, 0.17, 0.26}};
constexpr TileCost kGradient[] = {{256, 8, 1, 5.7, 4.63, 1.26, 0.95, 0.22, -1},
                                  {128, 4, 2, 4.0, 3.24, 0.67, 0.49, 0.21, -1},
                                  {64, 8, 1, 2.5, 0.0, 1.67, 0.88, 0.58, 0.17},
                                  {64, 4, 2, 2.9, 0.57, 0.98, 1.29, 0.35, 0.25},
                                  {64, 1, 8, 2.1, 3.64, 0.90, 1.51, 0.23, 0.40}};
constexpr TileCost kFewBits[] = {{256, 8, 1, 10.3, 0.43, 0.83, 1.50, 0.27, 0},
                                 {128, 4, 2, 7.0, 1.69, 0.48, 0.91, 0.26, 0},
                                 {64, 8, 1, 5.7, 0.29, 1.60, 1.34, 0.21, 0},
                                 {32, 8, 1, 5.3, 0.49, 1.04, 0.82, 0.18, 0}};

// Weights that one row block reads are loaded past the caches where all groups' are more than the last-level cache holds: 256 rows over 8
// groups of 14336 x 4096 168 -> 151 us (6.2 TB/s), 64 over 64 of 2048 x 8192 in 4 bits 65.8 -> 58.9, 16 over 32 of 2048 x 2048, other
// weights each call, 21.0 -> 19.4. Where the next call has the same few groups they could have stayed there (the last one, call after call:
// 17.6 -> 18.4); smaller weights may be there still: 14336 x 4096 in 4 bits, 16 rows, call after call 9.5 us, past the caches 10.0.
constexpr double kLastLevelCache = 256e6;

// Rows of weights that lie a power of two apart have the same place of K on few of the memory's channels, and workgroups that go through
// K in step ask for it together: so groups, and parts of the columns where groups are few, start at different K-tiles (group_turn_place).
// 2048 rows over 64 groups of 2048 x 2048 147 -> 115 us, 8192 over 64 147 -> 136, 16 over 32 21.8 -> 19.9, 16 rows by one of 14336 x 4096
// 26.7 -> 23.5; in 4 bits 64 over 64 of 2048 x 8192 67.6 -> 60.5. Rows other lengths apart lose nothing by it, so they are not told apart:
// 2048 over 64 of 2048 x 1536 93.1 -> 92.2, of 2048 x 2880 165.7 -> 165.5, 256 over 8 of 14336 x 5120 204.5 -> 204.3, 1000 rows by one
// of 4096 x 5000 92.9 -> 84.6. Groups of many rows gain nothing, and have their rows read at several K-tiles: 16384 over 4 of 4096 x
// 4096 475.7 -> 478.9, 8192 over 2 in 4 bits 101.4 -> 102.4. (Weights [K][N] are rows of other K-tiles.)
constexpr double kTurnedRows = 2048;

// Log2 of the parts of a group's columns that start apart. Groups start apart themselves; of one that has fewer than four row blocks (tile_at),
// an XCD has an eighth of the columns, of more row blocks or groups more of them, and workgroups of one XCD that start together share
// what its L2 holds: 8192 rows over 16 groups of 4096 x 4096 with eight parts 301 us, with one 295.
int log_turn_parts(int E, int T, int tile) {
  const long long blocks = ((long long)T + (long long)tile * E - 1) / ((long long)tile * E), runs = E * ((blocks + 3) / 4);
  return runs == 1 ? 3 : runs == 2 ? 2 : runs <= 4 ? 1 : 0;
}

double busy_groups(int E, int T) { return E > 1 ? E * -std::expm1(-(double)T / E) : 1.0; }
int tiles_across(int tile, int n) { return (int)(((long long)n + std::max(tile, 64) - 1) / std::max(tile, 64)); }

// wgs: workgroups with a tile of `tile`; k_tiles: of a tile; fits: a kernel's launch and counts can have this size. NULL: none can.
template <int N, typename WGS, typename FITS>
const TileCost *choose_tile(const TileCost (&costs)[N], bool even, int cus, double k_tiles, double mbytes, WGS wgs, FITS fits) {
  const TileCost *best = nullptr;
  double least = 0;
  for (const TileCost &c : costs) {
    if ((!even && c.any < 0) || !fits(c)) continue;
    const double there = wgs(c.tile) / ((double)cus * c.per_cu), rounds = std::max(1.0, 0.5 * (there + std::ceil(there)));
    const double steps = c.tile > 64 || c.waves == 1 ? k_tiles : std::ceil(k_tiles / c.waves);
    const double step = (c.step + c.full * std::min(1.0, there)) * (even ? 1.0 : 1.0 + c.any);
    const double x = rounds * (c.round + step * steps), y = mbytes * c.byte;
    const double t = c.start + std::max(x, y) + 0.15 * std::min(x, y);
    if (!best || t < least) best = &c, least = t;
  }
  return best;
}

std::string tile_name(const TileCost &c, bool even) {
  return std::to_string(c.tile) + (even ? "" : "_any") + (c.tile == 64 ? "_w" + std::to_string(c.waves) : "");
}

const char *dtype_name(int dtype) { return dtype == MTK_F16 ? "f16" : "bf16"; }

int plan_grouped(mtk_ctx *ctx, const mtk_grouped_desc *d_in, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  mtk_grouped_desc d = *d_in;
  int s = check_grouped(d);
  if (s != MTK_OK) return s;
  if (d.out_f32) return fail(MTK_ERR_INVALID, "out_f32 is for gradients");
  if ((s = check_ld(d.lda, d.K, "lda", &d.lda)) != MTK_OK || (s = check_ld(d.ldb, d.trans_b ? d.K : d.N, "ldb", &d.ldb)) != MTK_OK ||
      (s = check_ld(d.ldc, d.N, "ldc", &d.ldc)) != MTK_OK)
    return s;
  const long long b_rows = d.trans_b ? d.N : d.K, b_width = d.trans_b ? d.K : d.N;
  const uint64_t b_exact = 2 * ((uint64_t)(b_rows - 1) * (uint64_t)d.ldb + (uint64_t)b_width);
  if (b_exact > kMaxOperandBytes) return fail(MTK_ERR_UNSUPPORTED, "the weights of a group must be below 2 GiB");
  const int cus = ctx ? ctx->prop.multiProcessorCount : 256;
  const bool even = d.lda % 2 == 0 && d.ldb % 2 == 0;
  const double busy = busy_groups(d.E, d.T);
  auto count = [&](const TileCost &c) { return count_tiles(d.E, d.T, c.tile, c.waves, tiles_across(c.tile, d.N), cus); };
  const TileCost *chosen = choose_tile(kForward, even, cus, (d.K + 63) / 64, 2e-6 * (busy * d.N * d.K + (double)d.T * ((double)d.N + d.K)),
                                       [&](int t) { return std::max(busy, (double)d.T / t + 0.5 * busy) * tiles_across(t, d.N); },
                                       [&](const TileCost &c) { return count(c).fits; });
  if (!chosen) return fail(MTK_ERR_UNSUPPORTED, "%d groups of up to %d rows with N %d have too many tiles", d.E, d.T, d.N);
  const TileCost kind = *chosen;
  const int tile = kind.tile;
  mtk_grouped_kargs a{};
  a.E = d.E;
  a.T = d.T;
  a.N = d.N;
  a.K = d.K;
  a.lda = d.lda;
  a.ldb = d.ldb;
  a.ldc = d.ldc;
  a.b_stride = b_rows * d.ldb;
  a.b_exact = (uint32_t)b_exact;
  a.tiles_n = tiles_across(tile, d.N);
  a.k_tiles = (d.K + 63) / 64;
  a.has_bias = d.has_bias ? 1 : 0;
  a.b_once = 2.0 * d.E * d.N * d.K > kLastLevelCache ? 1 : 0;
  if (d.trans_b && d.T < kTurnedRows * busy && d.K >= 128) a.turns = group_turns_of(log_turn_parts(d.E, d.T, tile), a.tiles_n);
  const long long grid = count(kind).grid;
  std::unique_ptr<mtk_plan> p(new mtk_plan());
  p->ctx = ctx;
  p->kind = PLAN_GROUPED;
  p->grouped = d;
  p->align_a = p->align_b = even ? 4 : 2;
  const std::string name = std::string("mtk_grouped_") + dtype_name(d.dtype) + (d.trans_b ? "_nt_" : "_nn_") + tile_name(kind, even);
  add_launch(p.get(), name, grid, 64 * kind.waves, a);
  p->flops = 2.0 * d.T * d.N * d.K;
  p->bytes = 2.0 * ((double)d.T * (d.N + d.K) + (double)std::min(d.E, d.T) * d.N * d.K);
  char desc[256];
  snprintf(desc, sizeof desc, "grouped gemm %s E=%d T=%d N=%d K=%d b=%s bias=%d tile=%d grid=%lld", dtype_name(d.dtype), d.E, d.T,
           d.N, d.K, d.trans_b ? "nk" : "kn", a.has_bias, tile, grid);
  p->description = desc;
  return finish_plan(std::move(p), out);
}

int plan_grouped_grad(mtk_ctx *ctx, const mtk_grouped_desc *d_in, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  mtk_grouped_desc d = *d_in;
  int s = check_grouped(d);
  if (s != MTK_OK) return s;
  if (d.ldb) return fail(MTK_ERR_INVALID, "gradients of the weights are packed: ldb must be 0 (got %d)", d.ldb);
  if ((s = check_ld(d.lda, d.K, "lda", &d.lda)) != MTK_OK || (s = check_ld(d.ldc, d.N, "ldc", &d.ldc)) != MTK_OK) return s;
  for (int ld : {d.lda, d.ldc})
    if (2ull * (uint64_t)d.T * (uint64_t)ld > kMaxOperandBytes) return fail(MTK_ERR_UNSUPPORTED, "A and dC must be below 2 GiB");
  const int cus = ctx ? ctx->prop.multiProcessorCount : 256;
  const bool even = d.lda % 2 == 0 && d.ldc % 2 == 0;
  mtk_grouped_kargs a{};
  a.E = d.E;
  a.T = d.T;
  a.M = d.trans_b ? d.N : d.K;
  a.N = d.trans_b ? d.K : d.N;
  a.lda = d.trans_b ? d.ldc : d.lda;
  a.ldb = d.trans_b ? d.lda : d.ldc;
  auto wgs = [&](int tile) { return (long long)d.E * tiles_across(tile, a.M) * tiles_across(tile, a.N); };
  const long long bias_tiles = d.has_bias ? (long long)d.E * tiles_across(64, d.N) : 0, lead = (bias_tiles + 7) / 8 * 8;
  auto fits = [&](const TileCost &c) {
    if (c.tile == 64) return launches(wgs(64) + lead, 64 * c.waves);
    return wgs(c.tile) <= INT32_MAX && launches(bias_tiles, 512);
  };
  const double k_tiles = std::max(1.0, d.T / busy_groups(d.E, d.T) / 64);
  const TileCost *chosen = choose_tile(kGradient, even, cus, k_tiles, 1e-6 * ((d.out_f32 ? 4.0 : 2.0) * d.E * d.N * d.K + 2.0 * d.T * ((double)d.N + d.K)),
                                       [&](int t) { return (double)wgs(t); }, fits);
  if (!chosen) return fail(MTK_ERR_UNSUPPORTED, "%d groups with N %d and K %d have too many tiles", d.E, d.N, d.K);
  const TileCost kind = *chosen;
  const int tile = kind.tile;
  a.tiles_m = tiles_across(tile, a.M);
  a.tiles_n = tiles_across(tile, a.N);
  long long grid = tile_grid(tile, cus, wgs(tile));
  // Quarter tiles have the bias's sums in their launch: 1000 rows over 24 groups of 1023 x 520 33.2 -> 27.2 us, 2000 over 4 of 300 x 301
  // 13.1 -> 8.3, 1000 over 8 of 1024 x 512 13.9 -> 11.7. Large tiles are a persistent grid; beside them the bias has a launch of its own.
  const bool one_launch = d.has_bias && tile == 64;
  if (one_launch) {
    a.has_bias = d.trans_b ? 1 : 2;
    a.lead = (int)lead;
    grid += lead;
  }
  std::unique_ptr<mtk_plan> p(new mtk_plan());
  p->ctx = ctx;
  p->kind = PLAN_GROUPED_GRAD;
  p->grouped = d;
  p->align_a = p->align_b = even ? 4 : 2;
  const std::string head = std::string("mtk_grouped_") + dtype_name(d.dtype);
  const std::string name = head + "_grad_" + tile_name(kind, even);
  add_launch(p.get(), name, grid, 64 * kind.waves, a);
  if (d.has_bias && !one_launch) {
    mtk_grouped_kargs b{};
    b.E = d.E;
    b.T = d.T;
    b.N = d.N;
    b.lda = d.ldc;
    b.tiles_n = tiles_across(64, d.N);
    add_launch(p.get(), head + "_bias_grad", bias_tiles, 512, b);
    p->launches.back().role = ROLE_REDUCE;
  }
  p->flops = 2.0 * d.T * d.N * d.K;
  p->bytes = 2.0 * d.T * (d.N + d.K) + (d.out_f32 ? 4.0 : 2.0) * d.E * d.N * d.K;
  char desc[256];
  snprintf(desc, sizeof desc, "grouped gradient %s E=%d T=%d N=%d K=%d b=%s bias=%d out=%s tile=%d grid=%lld", dtype_name(d.dtype),
           d.E, d.T, d.N, d.K, d.trans_b ? "nk" : "kn", d.has_bias ? 1 : 0, d.out_f32 ? "f32" : "16", tile, grid);
  p->description = desc;
  return finish_plan(std::move(p), out);
}

// ------------------------------------------------------------------ rows in few bits

int check_mx_rows(long long R, long long K) {
  if (R <= 0 || K <= 0) return fail(MTK_ERR_INVALID, "R and K must be positive (got %lld, %lld)", R, K);
  if (K > kMaxWidth) return fail(MTK_ERR_UNSUPPORTED, "K above 2^22 is not supported (got %lld)", K);
  return MTK_OK;
}

// The launch that brings R rows into the format or back.
Launch mx_rows_launch(bool quantize, int R, int K, int ld, int dtype) {
  mtk_mx_rows_kargs a{};
  a.R = R;
  a.K = K;
  a.ld = ld;
  a.k_tiles = mx_k_tiles(K);
  const long long waves = ((long long)R + 3) / 4 * ((a.k_tiles + 1) / 2);  // 4 rows x 2 K-tiles each
  Launch l;
  l.name = std::string(quantize ? "mtk_mx_quantize_" : "mtk_mx_dequantize_") + dtype_name(dtype);
  l.grid = (unsigned)((waves + 3) / 4);
  set_args(l, a);
  return l;
}

int plan_mx_rows(mtk_ctx *ctx, const mtk_mx_rows_desc *d_in, bool quantize, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  mtk_mx_rows_desc d = *d_in;
  int s = check_mx_rows(d.R, d.K);
  if (s != MTK_OK) return s;
  if (d.dtype != MTK_F16 && d.dtype != MTK_BF16) return fail(MTK_ERR_INVALID, "dtype must be MTK_F16 or MTK_BF16");
  if ((s = check_ld(d.ld, d.K, "ld", &d.ld)) != MTK_OK) return s;
  if (!launches(((long long)d.R + 15) / 16 * ((mx_k_tiles(d.K) + 1) / 2), 256))
    return fail(MTK_ERR_UNSUPPORTED, "ceil(R / 16) x ceil(K / 512) has to be below 2^24 (got %d rows of %d)", d.R, d.K);
  std::unique_ptr<mtk_plan> p(new mtk_plan());
  p->ctx = ctx;
  p->kind = quantize ? PLAN_MX_QUANT : PLAN_MX_DEQUANT;
  p->mx_rows = d;
  p->launches.push_back(mx_rows_launch(quantize, d.R, d.K, d.ld, d.dtype));
  p->bytes = (double)d.R * (2.0 * d.K + 136.0 * mx_k_tiles(d.K));
  char desc[160];
  snprintf(desc, sizeof desc, "mx %s %s R=%d K=%d ld=%d grid=%u", quantize ? "quantize" : "dequantize", dtype_name(d.dtype), d.R, d.K, d.ld,
           p->launches[0].grid);
  p->description = desc;
  return finish_plan(std::move(p), out);
}

int plan_mx_gemm(mtk_ctx *ctx, const mtk_mx_gemm_desc *d_in, mtk_plan **out) {
  if (!d_in || !out) return fail(MTK_ERR_INVALID, "null descriptor or output");
  mtk_mx_gemm_desc d = *d_in;
  if (d.E < 0 || d.T <= 0 || d.N <= 0 || d.K <= 0)
    return fail(MTK_ERR_INVALID, "E must be 0 or more, T, N and K positive (got %d, %d, %d, %d)", d.E, d.T, d.N, d.K);
  if (d.N > kMaxWidth || d.K > kMaxWidth) return fail(MTK_ERR_UNSUPPORTED, "N and K above 2^22 are not supported (got %d, %d)", d.N, d.K);
  if (d.E > kMaxGroups) return fail(MTK_ERR_UNSUPPORTED, "E above 2^14 is not supported (got %d)", d.E);
  if (d.dtype != MTK_F16 && d.dtype != MTK_BF16) return fail(MTK_ERR_INVALID, "dtype must be MTK_F16 or MTK_BF16");
  if (!d.quantize_a && d.lda) return fail(MTK_ERR_INVALID, "lda is for 16-bit rows (quantize_a)");
  int s;
  if ((s = check_ld(d.lda, d.K, "lda", &d.lda)) != MTK_OK || (s = check_ld(d.ldc, d.N, "ldc", &d.ldc)) != MTK_OK) return s;
  const long long groups = d.E ? d.E : 1;
  const int k_tiles = mx_k_tiles(d.K);
  // scales of an operand are read with 32-bit offsets, 8 bytes a row and K-tile; and the rows' own launch can have so many
  constexpr long long kMostScales = (1ll << 28) - 32;
  if ((long long)d.T * k_tiles > kMostScales || groups * d.N > kMostScales / k_tiles)
    return fail(MTK_ERR_UNSUPPORTED, "T x ceil(K / 256) and E x N x ceil(K / 256) up to 2^28 - 32 are supported");
  mtk_mx_gemm_kargs a{};
  a.E = (int)groups;
  a.T = d.T;
  a.N = d.N;
  a.lda = d.lda;
  a.K = d.K;
  a.k_tiles = k_tiles;
  a.ldc = d.ldc;
  a.has_bias = d.has_bias ? 1 : 0;
  a.b_once = 136.0 * k_tiles * groups * d.N > kLastLevelCache ? 1 : 0;
  const int cus = ctx ? ctx->prop.multiProcessorCount : 256;
  const double busy = busy_groups((int)groups, d.T);
  auto count = [&](const TileCost &c) {
    TileCount n = count_tiles((int)groups, d.T, c.tile, c.waves, tiles_across(c.tile, d.N), cus);
    if (!d.E) n.grid = tile_grid(c.tile, cus, ((long long)d.T + c.tile - 1) / c.tile * tiles_across(c.tile, d.N));
    return n;
  };
  const TileCost *chosen = choose_tile(kFewBits, true, cus, k_tiles, 1e-6 * (0.53 * (busy * d.N * d.K + (double)d.T * d.K) + 2.0 * d.T * d.N),
                                       [&](int t) {
                                         return (d.E ? std::max(busy, (double)d.T / t + 0.5 * busy) : (double)((d.T + t - 1) / t)) * tiles_across(t, d.N);
                                       },
                                       [&](const TileCost &c) { return count(c).fits; });
  if (!chosen) return fail(MTK_ERR_UNSUPPORTED, "%lld groups of up to %d rows with N %d have too many tiles", groups, d.T, d.N);
  TileCost kind = *chosen;
  // Few rows are brought into the format by the product's own workgroups, each of them all that it needs, which takes longer than the
  // launch before it where a wavefront has many rows and K-tiles. 14336 x 4096: 1 row 7.7 us (with the launch 10.9), 8 rows 9.4 (11.3), 16
  // 11.3 (11.2); 2048 x 2048: 16 rows 7.1 (8.4); 4096 x 14336: 1 row 12.7 (13.8); 64 over 64 groups of 2048 x 8192 66.8 (60.3).
  const TileCost &few = kFewBits[3];
  const double per = d.E ? std::max(1.0, d.T / busy) : d.T, rounds = std::ceil(busy * tiles_across(32, d.N) / cus);
  const bool inside = d.quantize_a && d.T <= 32.0 * busy && std::ceil(per / 2) * std::ceil(k_tiles / 8.0) * rounds <= 8 && count(few).fits;
  if (inside) kind = few;
  const int tile = kind.tile;
  a.tiles_n = tiles_across(tile, d.N);
  if (d.T < kTurnedRows * busy && k_tiles > 1) a.turns = group_turns_of(log_turn_parts((int)groups, d.T, tile), a.tiles_n);
  const long long grid = count(kind).grid;
  std::unique_ptr<mtk_plan> p(new mtk_plan());
  p->ctx = ctx;
  p->kind = PLAN_MX_GEMM;
  p->mx_gemm = d;
  if (d.quantize_a && !inside) {
    p->launches.push_back(mx_rows_launch(true, d.T, d.K, d.lda, d.dtype));
    p->launches.back().role = ROLE_PERMUTE;
    p->scales_at = (mx_code_bytes(d.T, k_tiles) + 255) & ~(size_t)255;  // the scales
    p->workspace = p->scales_at + mx_scale_bytes(d.T, k_tiles);
  }
  const std::string name = std::string("mtk_mx_gemm_") + dtype_name(d.dtype) + "_" + std::to_string(tile) + (inside ? "q" : "");
  add_launch(p.get(), name, grid, 64 * kind.waves, a);
  p->flops = 2.0 * d.T * d.N * d.K;
  p->bytes = 136.0 * k_tiles * ((d.quantize_a ? 0.0 : d.T) + (double)std::min<long long>(groups, d.T) * d.N) + 2.0 * d.T * d.N +
             (d.quantize_a ? 2.0 * d.T * d.K : 0.0);
  char desc[256];
  snprintf(desc, sizeof desc, "mx gemm %s E=%d T=%d N=%d K=%d bias=%d quantize_a=%d tile=%d grid=%lld", dtype_name(d.dtype), d.E, d.T,
           d.N, d.K, a.has_bias, d.quantize_a ? 1 : 0, tile, grid);
  p->description = desc;
  return finish_plan(std::move(p), out);
}

// ------------------------------------------------------------------ run-time arguments

// What an operator reads or writes: n rows of `width` bytes, `step` bytes apart.
struct Rows {
  const char *name;
  const void *at;
  uint64_t n, width, step;
  uint64_t bytes() const { return (n - 1) * step + width; }
};
Rows flat(const char *name, const void *at, uint64_t bytes) { return {name, at, 1, bytes, bytes}; }

bool meet(const Rows &a, const Rows &b) {
  if (!a.at || !b.at || !a.width || !b.width || !overlap(a.at, a.bytes(), b.at, b.bytes())) return false;
  if (a.step != b.step || a.n < 2 || b.n < 2) return true;
  const Rows &x = (uintptr_t)a.at <= (uintptr_t)b.at ? a : b, &y = &x == &a ? b : a;
  const uint64_t apart = (uintptr_t)y.at - (uintptr_t)x.at, rows = apart / x.step, rest = apart % x.step;
  // a row of y starts `rest` bytes behind one of x, and ends before or behind the start of x's next
  return (rows < x.n && rest < x.width) || (rows + 1 < x.n && rest + y.width > x.step);
}

int check_overlaps(std::initializer_list<Rows> in, std::initializer_list<Rows> out) {
  for (const Rows *o = out.begin(); o != out.end(); ++o) {
    for (const Rows &x : in)
      if (meet(*o, x)) return fail(MTK_ERR_INVALID, "%s overlaps %s", o->name, x.name);
    for (const Rows *q = out.begin(); q != o; ++q)
      if (meet(*o, *q)) return fail(MTK_ERR_INVALID, "%s overlaps %s", o->name, q->name);
  }
  return MTK_OK;
}

Rows rows16(const char *name, const void *at, int n, int width, int ld) {
  return {name, at, (uint64_t)n, 2 * (uint64_t)width, 2 * (uint64_t)ld};
}

int check_grouped_args(const mtk_plan *p, const void *argset) {
  if (!argset) return fail(MTK_ERR_INVALID, "null arguments");
  auto workspace = [&](const void *ws) {
    return p->workspace && (!ws || !aligned(ws, 16))
               ? fail(MTK_ERR_INVALID, "this plan needs a 16-byte aligned workspace of %zu bytes", p->workspace)
               : MTK_OK;
  };
  int s;
  if (p->kind == PLAN_GROUPED) {
    const mtk_grouped_gemm_args *t = (const mtk_grouped_gemm_args *)argset;
    const mtk_grouped_desc &d = p->grouped;
    if (!t->A || !t->B || !t->C || !t->row_start) return fail(MTK_ERR_INVALID, "A, B, C and row_start must be non-null");
    if (d.has_bias && !t->bias) return fail(MTK_ERR_INVALID, "plan has a bias but bias is null");
    if (!aligned(t->A, p->align_a) || !aligned(t->B, p->align_b))
      return fail(MTK_ERR_INVALID, "A and B must be %u-byte aligned for this plan", p->align_a);
    if (!aligned(t->C, 2) || !aligned(t->bias, 2) || !aligned(t->row_start, 4))
      return fail(MTK_ERR_INVALID, "C and bias must be 2-byte, row_start 4-byte aligned");
    if ((s = workspace(t->workspace)) != MTK_OK) return s;
    const uint64_t b = 2 * (uint64_t)d.E * (uint64_t)(d.trans_b ? d.N : d.K) * (uint64_t)d.ldb;
    return check_overlaps({rows16("A", t->A, d.T, d.K, d.lda), flat("B", t->B, b - 2 * (uint64_t)(d.ldb - (d.trans_b ? d.K : d.N))),
                           flat("bias", d.has_bias ? t->bias : nullptr, 2 * (uint64_t)d.E * (uint64_t)d.N),
                           flat("row_start", t->row_start, 4 * ((uint64_t)d.E + 1))},
                          {rows16("C", t->C, d.T, d.N, d.ldc), flat("the workspace", t->workspace, p->workspace)});
  }
  if (p->kind == PLAN_GROUPED_GRAD) {
    const mtk_grouped_grad_args *t = (const mtk_grouped_grad_args *)argset;
    const mtk_grouped_desc &d = p->grouped;
    if (!t->A || !t->dC || !t->dB || !t->row_start) return fail(MTK_ERR_INVALID, "A, dC, dB and row_start must be non-null");
    if (d.has_bias && !t->dbias) return fail(MTK_ERR_INVALID, "plan has a bias but dbias is null");
    if (!aligned(t->A, p->align_a) || !aligned(t->dC, p->align_b))
      return fail(MTK_ERR_INVALID, "A and dC must be %u-byte aligned for this plan", p->align_a);
    if (!aligned(t->dB, 16) || !aligned(t->dbias, 4) || !aligned(t->row_start, 4))
      return fail(MTK_ERR_INVALID, "dB must be 16-byte, dbias and row_start 4-byte aligned");
    if ((s = workspace(t->workspace)) != MTK_OK) return s;
    const uint64_t size = d.out_f32 ? 4 : 2, groups = (uint64_t)d.E * (uint64_t)d.N;
    return check_overlaps({rows16("A", t->A, d.T, d.K, d.lda), rows16("dC", t->dC, d.T, d.N, d.ldc),
                           flat("row_start", t->row_start, 4 * ((uint64_t)d.E + 1))},
                          {flat("dB", t->dB, size * groups * (uint64_t)d.K), flat("dbias", d.has_bias ? t->dbias : nullptr, size * groups),
                           flat("the workspace", t->workspace, p->workspace)});
  }
  if (p->kind == PLAN_MX_QUANT || p->kind == PLAN_MX_DEQUANT) {
    const bool q = p->kind == PLAN_MX_QUANT;
    const mtk_mx_quantize_args *w = (const mtk_mx_quantize_args *)argset;
    const mtk_mx_dequantize_args *r = (const mtk_mx_dequantize_args *)argset;
    const void *rows = q ? w->src : r->dst, *codes = q ? w->codes : r->codes, *scales = q ? w->scales : r->scales;
    const mtk_mx_rows_desc &d = p->mx_rows;
    if (!rows || !codes || !scales) return fail(MTK_ERR_INVALID, "%s, codes and scales must be non-null", q ? "src" : "dst");
    if (!aligned(rows, 2)) return fail(MTK_ERR_INVALID, "%s must be 2-byte aligned", q ? "src" : "dst");
    if (!aligned(codes, 16) || !aligned(scales, 16)) return fail(MTK_ERR_INVALID, "codes and scales must be 16-byte aligned");
    const int kt = mx_k_tiles(d.K);
    const Rows x = rows16(q ? "src" : "dst", rows, d.R, d.K, d.ld), c = flat("codes", codes, mx_code_bytes(d.R, kt)),
               y = flat("scales", scales, mx_scale_bytes(d.R, kt));
    return q ? check_overlaps({x}, {c, y}) : check_overlaps({c, y}, {x});
  }
  const mtk_mx_gemm_args *t = (const mtk_mx_gemm_args *)argset;
  const mtk_mx_gemm_desc &d = p->mx_gemm;
  const int kt = mx_k_tiles(d.K);
  const int64_t b_rows = (int64_t)(d.E ? d.E : 1) * d.N;
  if (!t->A || !t->B || !t->b_scales || !t->C) return fail(MTK_ERR_INVALID, "A, B, b_scales and C must be non-null");
  if (d.quantize_a ? t->a_scales != nullptr : !t->a_scales)
    return fail(MTK_ERR_INVALID, d.quantize_a ? "a_scales must be NULL where the run quantises A" : "a_scales must be non-null");
  if (d.E ? !t->row_start : t->row_start != nullptr)
    return fail(MTK_ERR_INVALID, d.E ? "row_start must be non-null" : "row_start must be NULL without groups");
  if (d.has_bias && !t->bias) return fail(MTK_ERR_INVALID, "plan has a bias but bias is null");
  if (!aligned(t->A, d.quantize_a ? 2 : 16) || !aligned(t->a_scales, 16) || !aligned(t->B, 16) || !aligned(t->b_scales, 16))
    return fail(MTK_ERR_INVALID, "codes and scales must be 16-byte aligned (16-bit rows 2-byte)");
  if (!aligned(t->C, 2) || !aligned(t->bias, 2) || !aligned(t->row_start, 4))
    return fail(MTK_ERR_INVALID, "C and bias must be 2-byte, row_start 4-byte aligned");
  if ((s = workspace(t->workspace)) != MTK_OK) return s;
  return check_overlaps({d.quantize_a ? rows16("A", t->A, d.T, d.K, d.lda) : flat("A", t->A, mx_code_bytes(d.T, kt)),
                         flat("a_scales", t->a_scales, mx_scale_bytes(d.T, kt)), flat("B", t->B, mx_code_bytes(b_rows, kt)),
                         flat("b_scales", t->b_scales, mx_scale_bytes(b_rows, kt)),
                         flat("bias", d.has_bias ? t->bias : nullptr, 2 * (uint64_t)b_rows),
                         flat("row_start", t->row_start, 4 * ((uint64_t)d.E + 1))},
                        {rows16("C", t->C, d.T, d.N, d.ldc), flat("the workspace", t->workspace, p->workspace)});
}

// Writes the run-time pointers of a launch into `block`, a copy of its argument block.
void patch_grouped(const mtk_plan *p, const Launch &l, char *block, const void *argset) {
  if (p->kind == PLAN_GROUPED) {
    const mtk_grouped_gemm_args *t = (const mtk_grouped_gemm_args *)argset;
    mtk_grouped_kargs &a = *(mtk_grouped_kargs *)block;
    a.A = t->A;
    a.B = t->B;
    a.bias = t->bias;
    a.row_start = t->row_start;
    a.C = t->C;
  } else if (p->kind == PLAN_GROUPED_GRAD) {
    const mtk_grouped_grad_args *t = (const mtk_grouped_grad_args *)argset;
    mtk_grouped_kargs &a = *(mtk_grouped_kargs *)block;
    const bool bias = l.role == ROLE_REDUCE;
    a.A = bias || p->grouped.trans_b ? t->dC : t->A;
    a.B = bias ? nullptr : p->grouped.trans_b ? t->A : t->dC;
    a.row_start = t->row_start;
    a.bias = a.lead ? t->dbias : nullptr;
    void *out = bias ? t->dbias : t->dB;
    a.C = p->grouped.out_f32 ? nullptr : out;
    a.C32 = p->grouped.out_f32 ? (float *)out : nullptr;
  } else if (p->kind == PLAN_MX_GEMM && l.role == ROLE_MAIN) {
    const mtk_mx_gemm_args *t = (const mtk_mx_gemm_args *)argset;
    mtk_mx_gemm_kargs &a = *(mtk_mx_gemm_kargs *)block;
    const bool held = p->mx_gemm.quantize_a && p->workspace;  // the launch before has brought the rows into the format
    a.A = held ? t->workspace : t->A;
    a.a_scales = held ? (char *)t->workspace + p->scales_at : t->a_scales;
    a.B = t->B;
    a.b_scales = t->b_scales;
    a.bias = t->bias;
    a.row_start = t->row_start;
    a.C = t->C;
  } else {
    mtk_mx_rows_kargs &a = *(mtk_mx_rows_kargs *)block;
    if (p->kind == PLAN_MX_DEQUANT) {
      const mtk_mx_dequantize_args *t = (const mtk_mx_dequantize_args *)argset;
      a.codes = const_cast<void *>(t->codes);
      a.scales = const_cast<void *>(t->scales);
      a.dst = t->dst;
    } else if (p->kind == PLAN_MX_QUANT) {
      const mtk_mx_quantize_args *t = (const mtk_mx_quantize_args *)argset;
      a.src = t->src;
      a.codes = t->codes;
      a.scales = t->scales;
    } else {
      const mtk_mx_gemm_args *t = (const mtk_mx_gemm_args *)argset;
      a.src = t->A;
      a.codes = t->workspace;
      a.scales = (char *)t->workspace + p->scales_at;
    }
  }
}

// A run: argument blocks on the stack, nothing is allocated.
int run_grouped(const mtk_plan *p, PlanKind kind, const void *argset) {
  if (!p) return fail(MTK_ERR_INVALID, "null plan");
  if (p->kind != kind) return fail(MTK_ERR_INVALID, "the plan is of another operator");
  if (!p->ctx) return fail(MTK_ERR_INVALID, "plan was created without a context (dry plan)");
  const int s = check_grouped_args(p, argset);
  if (s != MTK_OK) return s;
  alignas(16) char block[256];
  HIP_TRY(hipSetDevice(p->ctx->device));
  for (const Launch &l : p->launches) {
    if (l.args.size() > sizeof block) return fail(MTK_ERR_INVALID, "argument block of %s too large", l.name.c_str());
    memcpy(block, l.args.data(), l.args.size());
    patch_grouped(p, l, block, argset);
    void *params[] = {block};
    const hipError_t e = hipModuleLaunchKernel(l.fn, l.grid, 1, 1, l.block, 1, 1, 0, p->ctx->stream, params, nullptr);
    if (e != hipSuccess) return fail(MTK_ERR_LAUNCH, "launch of %s failed: %s", l.name.c_str(), hipGetErrorString(e));
  }
  return MTK_OK;
}
