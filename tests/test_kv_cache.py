"""The paged key/value cache in few bits, on the host: what its plans refuse, which workgroup of an attention launch
does what (every step of every pair once, partial sums inside the workspace, whatever the lengths on the device hold),
and the numpy form of the format that the GPU tests compare with."""
import ctypes
import glob
import os
import shutil
import subprocess

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import kv

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
PAGES = dict(n_pages=20, page_size=16, max_pages=8)


def write_plan(**kw):
    a = {**dict(B=2, T=5, H_kv=2, D=64), **PAGES, **kw}
    return mtk.KvWritePlan(None, a.pop("B"), a.pop("T"), a.pop("H_kv"), a.pop("D"), **a)


def read_plan(**kw):
    a = {**dict(B=2, T=5, H_kv=2, D=64), **PAGES, **kw}
    return mtk.KvReadPlan(None, a.pop("B"), a.pop("T"), a.pop("H_kv"), a.pop("D"), **a)


def attn_plan(**kw):
    a = {**dict(B=2, T=5, H=8, H_kv=2, D=64), **PAGES, **kw}
    return mtk.KvAttentionPlan(None, a.pop("B"), a.pop("T"), a.pop("H"), a.pop("H_kv"), a.pop("D"), **a)


# ------------------------------------------------------------------ refusals

INVALID, UNSUPPORTED = mtk.MTK_ERR_INVALID, mtk.MTK_ERR_UNSUPPORTED
COMMON = [
    (dict(B=0), INVALID), (dict(T=0), INVALID), (dict(T=-1), INVALID), (dict(max_pages=0), INVALID),
    (dict(n_pages=0), INVALID), (dict(H_kv=0), INVALID), (dict(H_kv=-2), INVALID),
    (dict(D=0), UNSUPPORTED), (dict(D=12), UNSUPPORTED), (dict(D=264), UNSUPPORTED),
    (dict(page_size=8), INVALID), (dict(page_size=24), INVALID), (dict(page_size=2048), INVALID), (dict(page_size=0), INVALID),
    (dict(max_pages=(1 << 26) + 1), UNSUPPORTED),                    # more than 2^30 positions
    (dict(n_pages=(1 << 31) - 1, H_kv=1 << 20, H=1 << 20, D=256, page_size=1024), UNSUPPORTED),  # cannot be addressed
]


@pytest.mark.parametrize("make", [write_plan, read_plan, attn_plan])
@pytest.mark.parametrize("kw, status", COMMON, ids=str)
def test_plans_refuse(make, kw, status):
    kw = dict(kw)
    if make is not attn_plan:
        kw.pop("H", None)
    with pytest.raises(mtk.MtkError) as e:
        make(**kw)
    assert e.value.status == status and e.value.message


@pytest.mark.parametrize("make, kw, status", [
    (write_plan, dict(ld_k=120), INVALID), (write_plan, dict(ld_v=132), INVALID), (write_plan, dict(ld_k=-128), INVALID),
    (read_plan, dict(ld_k=8), INVALID), (read_plan, dict(ld_v=129), INVALID),
    (write_plan, dict(H_kv=(1 << 20) + 1), UNSUPPORTED), (read_plan, dict(T=(1 << 31) - 1, H_kv=1 << 20), UNSUPPORTED),
    (attn_plan, dict(H=7), INVALID), (attn_plan, dict(H=0), INVALID), (attn_plan, dict(H=-2), INVALID),
    (attn_plan, dict(S_q=6), INVALID), (attn_plan, dict(S_q=-1), INVALID),
    (attn_plan, dict(ld_q=504), INVALID), (attn_plan, dict(ld_q=516), INVALID),
    (attn_plan, dict(T=1 << 26, B=1), UNSUPPORTED),                  # T x H
    (attn_plan, dict(B=1 << 22, T=1 << 22), UNSUPPORTED),            # row blocks
    (attn_plan, dict(B=1 << 20, T=1 << 20, S_q=1, max_pages=1 << 20), UNSUPPORTED),  # row blocks x steps
], ids=str)
def test_plans_refuse_more(make, kw, status):
    with pytest.raises(mtk.MtkError) as e:
        make(**kw)
    assert e.value.status == status and e.value.message


def test_bad_format_and_null_pointers():
    L = mtk.lib()
    d = mtk.KvDesc(B=1, T=1, H=1, H_kv=1, D=64, n_pages=1, page_size=16, max_pages=1, format=2, dtype=mtk.F16)
    h, n = ctypes.c_void_p(), ctypes.c_size_t()
    for fn in (L.mtk_kv_write_plan, L.mtk_kv_read_plan, L.mtk_kv_attn_plan):
        assert fn(None, ctypes.byref(d), ctypes.byref(h)) == INVALID and b"format" in L.mtk_last_error()
        assert fn(None, None, ctypes.byref(h)) == INVALID
        assert fn(None, ctypes.byref(d), None) == INVALID
    assert L.mtk_kv_cache_bytes(ctypes.byref(d), ctypes.byref(n)) == INVALID
    assert L.mtk_kv_cache_bytes(None, ctypes.byref(n)) == INVALID
    d.format, d.dtype = mtk.KV_FP8, mtk.F32
    for fn in (L.mtk_kv_write_plan, L.mtk_kv_read_plan, L.mtk_kv_attn_plan):
        assert fn(None, ctypes.byref(d), ctypes.byref(h)) == INVALID and b"dtype" in L.mtk_last_error()
    assert L.mtk_kv_cache_bytes(ctypes.byref(d), None) == INVALID
    with pytest.raises(KeyError):
        write_plan(format="fp6")


def test_dry_plans_and_plans_of_another_kind_refuse_to_run():
    p = 0x1000
    for plan, args in ((write_plan(), (p, p, p, p, p, p)), (read_plan(), (p, p, p, p, p, p)), (attn_plan(), (p, p, p, p, p, p))):
        with pytest.raises(mtk.MtkError) as e:
            plan.run(*args)
        assert e.value.status == INVALID and "context" in e.value.message
    L, w = mtk.lib(), write_plan()
    args = mtk.KvAttnArgs()
    assert L.mtk_kv_attn_run(w.handle, ctypes.byref(args)) == INVALID and b"not a plan for" in L.mtk_last_error()
    assert L.mtk_kv_read_run(w.handle, ctypes.byref(mtk.KvReadArgs())) == INVALID
    assert L.mtk_kv_write_run(None, ctypes.byref(mtk.KvWriteArgs())) == INVALID
    gemm = mtk.GemmPlan(None, 64, 64, 64)
    assert L.mtk_kv_write_run(gemm.handle, ctypes.byref(mtk.KvWriteArgs())) == INVALID


# ------------------------------------------------------------------ sizes and kernel choice

@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("H_kv, D, page", [(1, 8, 16), (3, 80, 64), (8, 128, 16), (2, 256, 1024)])
def test_cache_bytes(fmt, H_kv, D, page):
    assert mtk.kv_cache_bytes(7, page, H_kv, D, fmt) == kv.Cache(7, page, H_kv, D, fmt, "f16").bytes.size


def test_kernel_choice():
    few = attn_plan(B=64, T=64, H=32, H_kv=8, D=128, max_pages=1000, S_q=1, format="fp4")
    assert "mtk_kv_attend_fp4_d128_r1_f16 mtk_kv_join" in few.describe() and few.workspace_bytes > 0
    short = attn_plan(B=4, T=4, H=32, H_kv=8, D=128, max_pages=100, S_q=1)
    assert short.describe().endswith("kernels: mtk_kv_attend_fp4_d128_r1_w16_f16") and short.workspace_bytes == 0
    drafts = attn_plan(B=8, T=40, H=32, H_kv=8, D=96, max_pages=1000, S_q=5, format="fp8", dtype="bf16")
    assert "mtk_kv_attend_fp8_d128_r2_bf16" in drafts.describe()
    mixed = attn_plan(B=8, T=2000, H=32, H_kv=8, D=200, max_pages=1000, dtype="bf16")
    assert "mtk_kv_attend_fp4_d256_r1_bf16" in mixed.describe() and "mtk_kv_prefill_fp4_d256_bf16" in mixed.describe()


# ------------------------------------------------------------------ the runtime and the schedule, in C++

DRIVER = r"""
#include "runtime.cpp"
#include <map>
#include <random>
#include <set>

static int failures = 0;
#define CHECK(x, ...) do { if (!(x)) { printf("failed: %s: ", #x); printf(__VA_ARGS__); printf("\n"); if (++failures > 20) exit(1); } } while (0)

// What the kernels of a launch do with a batch (kv_device.hpp: lay, at), with the functions that they share with the
// host: how often each step of each pair is taken, and the places of partial sums.
static void schedule(const mtk_kv_attn_kargs &k, unsigned grid, const std::vector<int> &start, const std::vector<int> &len,
                     bool sane) {
  struct Pairs { kv_share h; int base, length; };
  std::vector<Pairs> seqs;
  int64_t work = 0, own = 0;
  for (int b = 0; b < k.B; ++b) {
    const kv_seq s = kv_sequence(start[b], start[b + 1], len[b], k.T, k.max_pages, k.page_shift);
    CHECK(s.first >= 0 && s.rows >= 0 && s.first + s.rows <= k.T && s.keys >= 0 && s.keys <= (k.max_pages << k.page_shift), "%d", b);
    seqs.push_back({kv_blocks(s, k.S_q, k.G, k.rows_shift, k.step_shift, k.rows_above, k.rows_most), 0, 0});
    const kv_share &h = seqs.back().h;
    work += (int64_t)h.blocks * k.H_kv * h.steps;
    own += (int64_t)h.blocks * k.H_kv * kv_own(h, k.least);
  }
  CHECK(work <= INT32_MAX && own * k.least <= INT32_MAX, "work %lld own %lld", (long long)work, (long long)own);
  kv_cut cut;
  if (k.by_pair) {
    int64_t pairs = 0;
    for (auto &s : seqs) pairs += s.h.blocks * k.H_kv;
    const int most = (int)((((int64_t)k.max_pages << k.page_shift) + (1 << k.step_shift) - 1) >> k.step_shift);
    int hi = kv_each_of_pairs((int)work, (int)pairs, k.units, k.least, most);
    auto wgs_of = [&](int each) {
      int64_t n = 0;
      for (auto &s : seqs) n += s.h.blocks * (int64_t)k.H_kv * ((s.h.steps + each - 1) / each);
      return n;
    };
    CHECK(wgs_of(hi) <= std::max<int64_t>(k.units, pairs), "each %d", hi);
    if (k.B <= 64 && kv_pairs_split((int)work, (int)pairs, k.units))
      for (int lo = std::min(hi, std::max<int>(k.least, (work + k.units - 1) / k.units)); lo < hi;) {
        const int mid = (lo + hi) >> 1;
        wgs_of(mid) <= k.units ? hi = mid : lo = mid + 1;
      }
    cut = {hi, 1};
  }
  else cut = kv_cut_of((int)work, (int)own, k.units, k.least);
  if (k.whole && !k.by_pair) {  // by the workgroup's number
    CHECK(grid == (unsigned)(k.B * k.H_kv), "grid %u", grid);
    for (auto &s : seqs) CHECK(s.h.blocks <= 1, "blocks %d", s.h.blocks);
    return;
  }
  int64_t total = 0;
  for (auto &s : seqs) {
    s.length = kv_length(s.h, cut);
    s.base = (int)total;
    total += (int64_t)s.h.blocks * k.H_kv * s.length;
  }
  CHECK(total <= INT32_MAX, "line of %lld", (long long)total);
  const int64_t wgs = (total + cut.each - 1) / cut.each;
  if (!sane && k.by_pair) return;  // rows claimed twice: workgroups past the grid are not there, and write nothing
  CHECK(wgs <= (int64_t)grid, "%lld workgroups, grid %u", (long long)wgs, grid);
  if (k.places && !k.by_pair) CHECK(wgs <= k.places, "%lld workgroups, %d places", (long long)wgs, k.places);
  for (auto &s : seqs)
    for (int p = 0; p < s.h.blocks * k.H_kv; ++p) {
      const int64_t at = s.base + (int64_t)p * s.length;
      if (k.by_pair) CHECK(at % cut.each == 0 && s.length % cut.each == 0, "pair at %lld", (long long)at);
      if (k.by_pair && s.h.steps > cut.each) CHECK((at + s.h.steps - 1) / cut.each < k.places, "place of %lld", (long long)at);
      if (!k.places) CHECK(at / cut.each == (at + s.h.steps - 1) / cut.each, "a pair of several workgroups without a workspace");
      CHECK(s.length >= s.h.steps && s.length < s.h.steps + cut.each, "length %d of %d", s.length, s.h.steps);
      // at most two pairs of a workgroup are shared: its first and its last
      const int64_t w0 = at / cut.each, w1 = (at + s.h.steps - 1) / cut.each;
      if (w0 != w1) CHECK(at % cut.each == 0 || at / cut.each * cut.each != at, "%lld", (long long)at);
    }
}

static size_t part_rows(const mtk_kv_attn_kargs &k) {
  return (size_t)k.places * (k.by_pair ? 1 : 2) * (1u << k.rows_shift);
}

int main() {
  std::mt19937 rng(11);
  auto log = [&](int lo, int hi) { return (int)(lo * std::pow((double)hi / lo, std::uniform_real_distribution<>(0, 1)(rng))); };
  std::set<std::string> names;
  int plans = 0, split = 0;
  for (int n = 0; n < 30000; ++n) {
    mtk_kv_desc d{};
    const int groups[] = {1, 1, 2, 3, 4, 8, 16, 71};
    d.B = log(1, 300), d.H_kv = log(1, 33), d.H = d.H_kv * groups[rng() % 8], d.D = 8 * log(1, 33), d.T = log(1, 5000);
    d.S_q = rng() % 2 ? 0 : std::min(d.T, log(1, 600));
    d.page_size = 16 << rng() % 7, d.max_pages = log(1, 4000), d.n_pages = log(1, 100000), d.format = rng() % 2, d.dtype = rng() % 2;
    d.causal = rng() % 2;
    mtk_plan *p = nullptr;
    if (mtk_kv_attn_plan(nullptr, &d, &p) != MTK_OK) continue;
    ++plans;
    size_t used = 0;
    CHECK(p->launches.size() >= 1 && p->launches.size() <= 4, "%zu launches", p->launches.size());
    const bool sane = rng() % 4 != 0;
    std::vector<int> start(d.B + 1), len(d.B);
    const int64_t cap = (int64_t)d.max_pages * d.page_size;
    for (int b = 0; b <= d.B; ++b) start[b] = sane ? (int)(rng() % (d.T + 1)) : (int)rng();
    if (sane) std::sort(start.begin(), start.end());
    for (int b = 0; b < d.B; ++b) len[b] = rng() % 5 == 0 ? (sane ? 0 : (int)rng()) : log(1, (int)cap + 1);
    const mtk_kv_attn_kargs *before = nullptr;  // whose partial sums are not joined yet
    for (Launch &l : p->launches) {
      names.insert(l.name);
      const mtk_kv_attn_kargs &k = args_of<mtk_kv_attn_kargs>(l);
      if (l.name.find("join") != std::string::npos) {  // after its launch
        CHECK(before && before->places > 0 && memcmp(&k, before, sizeof k) == 0, "%s", p->description.c_str());
        before = nullptr;
        continue;
      }
      unsigned grid = l.grid;
      if (l.name.find("prefill") != std::string::npos) {  // joins the sums of the launch before it, if there are any
        const mtk_kv_prefill_kargs &both = args_of<mtk_kv_prefill_kargs>(l);
        CHECK((both.joins > 0) == (before && before->places > 0), "%d joins", both.joins);
        if (both.joins) CHECK(memcmp(&both.join, before, sizeof k) == 0, "%s", p->description.c_str());
        grid -= both.joins;
        before = nullptr;
      }
      CHECK(!before || before->places == 0, "%s", p->description.c_str());
      before = k.places ? &k : nullptr;
      CHECK(!k.places || (unsigned)k.places == grid || (k.by_pair && (unsigned)k.places < grid), "%d places", k.places);
      if (k.places) {  // partial sums, then their statistics, one launch's after another's
        const size_t rows = part_rows(k);
        CHECK((size_t)k.part == used && used % 16 == 0 && (size_t)k.part_ml % 8 == 0, "%s", p->description.c_str());
        CHECK((size_t)k.part + rows * k.part_ld * 4 <= (size_t)k.part_ml, "%s", p->description.c_str());
        used = (size_t)k.part_ml + rows * 8;
        CHECK(k.part_ld >= d.D && k.part_ld % 4 == 0, "%d", k.part_ld);
        ++split;
      }
      schedule(k, grid, start, len, sane);
    }
    CHECK(!before, "%s", p->description.c_str());
    CHECK(used <= p->workspace, "%zu of %zu", used, p->workspace);
    mtk_plan_destroy(p);
  }
  for (int n = 0; n < 2000; ++n) {  // rows written and read: a wavefront for each 64 items of each few rows
    mtk_kv_desc d{};
    d.B = log(1, 300), d.H_kv = log(1, 65), d.D = 8 * log(1, 33), d.T = log(1, 100000), d.page_size = 16 << rng() % 7, d.max_pages = 1000;
    d.n_pages = 1000, d.format = rng() % 2, d.dtype = rng() % 2;
    for (auto make : {mtk_kv_write_plan, mtk_kv_read_plan}) {
      mtk_plan *p = nullptr;
      if (make(nullptr, &d, &p) != MTK_OK) return printf("refused: %s\n", mtk_last_error()), 1;
      names.insert(p->launches[0].name);
      const mtk_kv_move_kargs &a = args_of<mtk_kv_move_kargs>(p->launches[0]);
      CHECK((int64_t)a.parts * 64 >= 8LL * d.H_kv * a.blocks && a.rows_per_wave <= 64, "%d parts", a.parts);
      CHECK(4LL * p->launches[0].grid * a.rows_per_wave >= (int64_t)d.T * a.parts, "grid %u", p->launches[0].grid);
      for (int i = 0; i < 8 * d.H_kv * a.blocks; ++i)  // the kernels' division by the blocks of a head
        CHECK((a.mul_blocks ? (int)(((uint64_t)(i >> 2) * a.mul_blocks) >> 32) : i >> 2) == (i >> 2) / a.blocks, "%d", i);
      mtk_plan_destroy(p);
    }
  }

  // ---- pages: entries out of range, positions past the table, before it, and the largest
  const int32_t row[4] = {3, -1, 7, INT32_MIN};
  CHECK(kv_page(row, 0, 8, 4, 4) == 3 && kv_page(row, 15, 8, 4, 4) == 3 && kv_page(row, 16, 8, 4, 4) == -1, " ");
  CHECK(kv_page(row, 32, 8, 4, 4) == 7 && kv_page(row, 32, 7, 4, 4) == -1 && kv_page(row, 48, 8, 4, 4) == -1, " ");
  CHECK(kv_page(row, 64, 8, 4, 4) == -1 && kv_page(row, -1, 8, 4, 4) == -1 && kv_page(row, INT64_MAX, 8, 4, 4) == -1, " ");
  CHECK(kv_page(row, INT32_MIN, 8, 4, 4) == -1, " ");
  const int any[] = {INT32_MIN, -1, 0, 1, 63, 64, 65, INT32_MAX};
  for (int a : any) for (int b : any) for (int n : any) {
    const kv_seq s = kv_sequence(a, b, n, 64, 4, 4);
    CHECK(s.first >= 0 && s.rows >= 0 && s.first + s.rows <= 64 && s.keys >= 0 && s.keys <= 64 && s.bad == (n > 64), "%d %d %d", a, b, n);
  }

  // ---- pointers, as a run checks them
  mtk_kv_desc d{};
  d.B = 2, d.T = 40, d.H = 8, d.H_kv = 2, d.D = 64, d.n_pages = 20, d.page_size = 16, d.max_pages = 600, d.dtype = MTK_F16;
  mtk_plan *w = nullptr, *r = nullptr, *t = nullptr;
  if (mtk_kv_write_plan(nullptr, &d, &w) || mtk_kv_read_plan(nullptr, &d, &r) || mtk_kv_attn_plan(nullptr, &d, &t)) return puts(mtk_last_error()), 1;
  char *at = (char *)0x100000000ull;
  const size_t cache = kv_cache_size(d), rows = 2 * 40 * 2 * 64, q = 2 * 40 * 8 * 64;
  int32_t *ints = (int32_t *)(at + (1 << 28));
  const mtk_kv_write_args ok{at, at + rows, at + 2 * rows, ints, ints, ints};
  CHECK(check_kv_args(w, &ok) == MTK_OK, "%s", mtk_last_error());
  auto bad = [&](const mtk_plan *p, const void *x, const char *says) {
    CHECK(check_kv_args(p, x) == MTK_ERR_INVALID && strstr(mtk_last_error(), says), "%s: %s", says, mtk_last_error());
  };
  bad(w, nullptr, "null arguments");
  for (int i = 0; i < 6; ++i) {  // each pointer null, and off by a byte
    mtk_kv_write_args x = ok;
    (&x.K)[i] = nullptr;
    bad(w, &x, "non-null");
    x = ok;
    (&x.K)[i] = (char *)(&ok.K)[i] + 1;
    bad(w, &x, "aligned");
  }
  mtk_kv_write_args over = ok;
  over.cache = at + rows - 16;
  bad(w, &over, "overlaps the cache");
  over = ok, over.cache = at + 3 * rows, over.V = at + 3 * rows + cache - 16;
  bad(w, &over, "overlaps the cache");
  over.V = at + 3 * rows + (cache + 15) / 16 * 16;
  CHECK(check_kv_args(w, &over) == MTK_OK, "%s", mtk_last_error());
  const mtk_kv_read_args rd{at, ints, ints, ints, at + cache, at + cache + rows};
  CHECK(check_kv_args(r, &rd) == MTK_OK, "%s", mtk_last_error());
  mtk_kv_read_args rx = rd;
  rx.K = at;
  bad(r, &rx, "overlaps the cache");
  rx = rd, rx.V = rd.K;
  bad(r, &rx, "the same rows");
  CHECK(t->workspace > 0, " ");
  const mtk_kv_attn_args ta{at, at + q, ints, ints, ints, at + q + (1 << 24), nullptr, at + (1 << 26)};
  CHECK(check_kv_args(t, &ta) == MTK_OK, "%s", mtk_last_error());
  mtk_kv_attn_args tx = ta;
  tx.O = at + q - 16;
  bad(t, &tx, "O overlaps Q");
  tx = ta, tx.O = nullptr;
  bad(t, &tx, "non-null");
  tx = ta, tx.Q = at + 8;
  bad(t, &tx, "aligned");
  tx = ta, tx.lse = (float *)(at + 2);
  bad(t, &tx, "lse");
  tx = ta, tx.workspace = nullptr;
  bad(t, &tx, "workspace");
  tx = ta, tx.workspace = at + 8;
  bad(t, &tx, "workspace");
  tx = ta, tx.O = at + q + 16;
  bad(t, &tx, "O overlaps the cache");
  tx = ta, tx.workspace = (void *)ta.O;
  bad(t, &tx, "the workspace overlaps O");

  if (plans < 15000 || split < 5000) return printf("%d plans, %d split\n", plans, split), 1;
  if (failures) return 1;
  for (auto &x : names) printf("%s\n", x.c_str());
  return 0;
}
"""


def test_schedule_and_arguments(tmp_path):
    scratch_obj = os.path.join(mtk.LIB_DIR, "scratch.o")
    if shutil.which("g++") is None or not os.path.exists(scratch_obj):
        pytest.skip("needs g++ and a built library (python -m example_matmul_metal4_amd.build)")
    src, exe = tmp_path / "kv.cpp", tmp_path / "kv"
    src.write_text(DRIVER)
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROCM}/include", f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), scratch_obj, f"-L{ROCM}/lib",
                        "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-ldl", "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    names = r.stdout.split()
    built = b"".join(open(f, "rb").read() for f in glob.glob(os.path.join(mtk.LIB_DIR, "mtk_kv_*.hsaco")))
    assert [n for n in names if n.encode() + b"\0" not in built] == []
    # and none that no plan runs
    import re
    have = {n.decode() for n in re.findall(rb"mtk_kv_[a-z0-9_]+(?=\.kd\0)", built)}
    assert have == set(names), have ^ set(names)


# ------------------------------------------------------------------ the numpy form

@pytest.mark.parametrize("fmt, most", [("fp4", 6.0), ("fp8", 448.0)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_format_in_numpy(fmt, most, dtype):
    rng = np.random.default_rng(3)
    x = kv.bits_of(rng.standard_normal((500, 64)) * 2.0 ** rng.integers(-12, 9, (500, 1)), dtype)
    codes, scales = kv.quantise(x, fmt, dtype)
    v, w = kv.to_f64(x, dtype), kv.dequantise(codes, scales, fmt)
    top = np.abs(v.reshape(500, 2, 32)).max(-1)
    s = 2.0 ** (scales.astype(np.float64) - 127)
    assert (top <= most * s).all() and ((top > most * s / 2) | (scales == 1)).all()  # the smallest power of two
    # half a step: of 2 (4 to 6) and below, relative to the scale; e4m3: 2^-4 of the value, or of the least normal number
    v3, w3 = v.reshape(500, 2, 32), w.reshape(500, 2, 32)
    step = s[..., None] * (1.0 if fmt == "fp4" else 0) + np.maximum(np.abs(v3) * 2.0 ** -4, s[..., None] * 2.0 ** -10) * (fmt == "fp8")
    assert (np.abs(v3 - w3) <= step).all()
    again, s2 = kv.quantise(kv.bits_of(w, "bf16"), fmt, "bf16")  # bf16 holds every value
    assert np.array_equal(kv.dequantise(again, s2, fmt), w)  # what was read back is written unchanged
    size = np.linalg.norm(v3 - w3) / np.linalg.norm(v3)
    assert size < (0.13 if fmt == "fp4" else 0.03)
