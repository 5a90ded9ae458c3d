"""Products grouped by expert and in 4 bits, on the host: what their plans and runs refuse, which kernels they choose (each is
built, and none is that no plan chooses), the arithmetic that places groups and tiles, and the numpy forms that the GPU tests
compare with."""
import ctypes
import glob
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
INVALID, UNSUPPORTED = mtk.MTK_ERR_INVALID, mtk.MTK_ERR_UNSUPPORTED
MOST = (1 << 31) - 1


def product(**kw):
    a = {**dict(E=3, T=50, N=64, K=96), **kw}
    return mtk.GroupedGemmPlan(None, a.pop("E"), a.pop("T"), a.pop("N"), a.pop("K"), **a)


def gradient(**kw):
    a = {**dict(E=3, T=50, N=64, K=96), **kw}
    return mtk.GroupedGradPlan(None, a.pop("E"), a.pop("T"), a.pop("N"), a.pop("K"), **a)


def quantise(**kw):
    a = {**dict(R=50, K=96), **kw}
    return mtk.MxQuantizePlan(None, a.pop("R"), a.pop("K"), **a)


def dequantise(**kw):
    a = {**dict(R=50, K=96), **kw}
    return mtk.MxDequantizePlan(None, a.pop("R"), a.pop("K"), **a)


def few_bits(**kw):
    a = {**dict(T=50, N=64, K=96), **kw}
    return mtk.MxGemmPlan(None, a.pop("T"), a.pop("N"), a.pop("K"), **a)


# ------------------------------------------------------------------ refusals

@pytest.mark.parametrize("make, kw, status", [
    *[(m, {n: v}, INVALID) for m in (product, gradient) for n in "ETNK" for v in (0, -1, -MOST - 1)],
    *[(m, {n: (1 << 22) + 1}, UNSUPPORTED) for m in (product, gradient) for n in "NK"],
    *[(m, dict(E=(1 << 14) + 1), UNSUPPORTED) for m in (product, gradient)],
    *[(m, {n: v}, INVALID) for m in (product, gradient) for n in ("lda", "ldc") for v in (63, -96)],
    *[(m, {n: (1 << 22) + 1}, UNSUPPORTED) for m in (product, gradient) for n in ("lda", "ldc")],
    (product, dict(ldb=95), INVALID), (product, dict(ldb=63, trans_b=False), INVALID), (product, dict(ldb=-1), INVALID),
    (product, dict(N=1 << 20, K=1 << 10), UNSUPPORTED), (product, dict(N=1 << 10, K=1 << 20, trans_b=False), UNSUPPORTED),  # 2 GiB a group
    (product, dict(T=MOST), UNSUPPORTED), (product, dict(T=MOST, E=1, N=1, K=1), UNSUPPORTED), (product, dict(E=1 << 14, T=MOST, N=1 << 20, K=1), UNSUPPORTED),
    (gradient, dict(T=MOST), UNSUPPORTED), (gradient, dict(T=1 << 24, lda=128), UNSUPPORTED), (gradient, dict(T=1 << 24, ldc=128), UNSUPPORTED),
    (gradient, dict(E=1 << 14, T=1, N=1 << 20, K=1 << 20), UNSUPPORTED),
    *[(m, {n: v}, INVALID) for m in (quantise, dequantise) for n in "RK" for v in (0, -1)],
    *[(m, dict(K=(1 << 22) + 1), UNSUPPORTED) for m in (quantise, dequantise)],
    *[(m, dict(ld=v), INVALID) for m in (quantise, dequantise) for v in (95, -96)],
    *[(m, dict(ld=(1 << 22) + 1), UNSUPPORTED) for m in (quantise, dequantise)],
    *[(m, dict(R=MOST), UNSUPPORTED) for m in (quantise, dequantise)],
    *[(few_bits, {n: v}, INVALID) for n in "TNK" for v in (0, -1)], (few_bits, dict(E=-1), INVALID),
    (few_bits, dict(E=(1 << 14) + 1), UNSUPPORTED), (few_bits, dict(N=(1 << 22) + 1), UNSUPPORTED), (few_bits, dict(K=(1 << 22) + 1), UNSUPPORTED),
    (few_bits, dict(lda=96), INVALID), (few_bits, dict(lda=95, quantize_a=True), INVALID), (few_bits, dict(ldc=63), INVALID),
    (few_bits, dict(ldc=(1 << 22) + 1), UNSUPPORTED), (few_bits, dict(T=MOST), UNSUPPORTED), (few_bits, dict(T=1 << 20, K=1 << 17), UNSUPPORTED),
    (few_bits, dict(E=1 << 14, N=1 << 20), UNSUPPORTED), (few_bits, dict(N=1 << 22, K=1 << 22), UNSUPPORTED),
], ids=lambda x: getattr(x, "__name__", str(x)))
def test_plans_refuse(make, kw, status):
    with pytest.raises(mtk.MtkError) as e:
        make(**kw)
    assert e.value.status == status and e.value.message


def test_descriptors_that_are_none():
    L, h, n = mtk.lib(), ctypes.c_void_p(), ctypes.c_size_t()
    for fn, d in ((L.mtk_grouped_gemm_plan, mtk.GroupedDesc(E=1, T=1, N=1, K=1)), (L.mtk_grouped_grad_plan, mtk.GroupedDesc(E=1, T=1, N=1, K=1)),
                  (L.mtk_mx_quantize_plan, mtk.MxRowsDesc(R=1, K=1)), (L.mtk_mx_dequantize_plan, mtk.MxRowsDesc(R=1, K=1)),
                  (L.mtk_mx_gemm_plan, mtk.MxGemmDesc(T=1, N=1, K=1))):
        for bad in (mtk.F32, 3, -1):
            d.dtype = bad
            assert fn(None, ctypes.byref(d), ctypes.byref(h)) == INVALID and b"dtype" in L.mtk_last_error()
        assert fn(None, None, ctypes.byref(h)) == INVALID
        assert fn(None, ctypes.byref(d), None) == INVALID
    d = mtk.GroupedDesc(E=1, T=1, N=1, K=1, dtype=mtk.F16, out_f32=1)
    assert L.mtk_grouped_gemm_plan(None, ctypes.byref(d), ctypes.byref(h)) == INVALID and b"out_f32" in L.mtk_last_error()
    d = mtk.GroupedDesc(E=1, T=1, N=1, K=1, dtype=mtk.F16, ldb=1)
    assert L.mtk_grouped_grad_plan(None, ctypes.byref(d), ctypes.byref(h)) == INVALID and b"ldb" in L.mtk_last_error()
    for R, K in ((0, 1), (1, 0), (-1, 5), (1, (1 << 22) + 1)):
        assert L.mtk_mx_bytes(R, K, ctypes.byref(n), ctypes.byref(n)) in (INVALID, UNSUPPORTED) and L.mtk_last_error()


def test_dry_plans_and_plans_of_another_kind_refuse_to_run():
    p = 0x1000
    plans = [(product(), (p, p, None, p, p)), (gradient(), (p, p, p, p)), (quantise(), (p, p, p)), (dequantise(), (p, p, p)),
             (few_bits(), (p, p, p, p, None, None, p))]
    for plan, args in plans:
        with pytest.raises(mtk.MtkError) as e:
            plan.run(*args)
        assert e.value.status == INVALID and "context" in e.value.message
    L = mtk.lib()
    runs = [("mtk_grouped_gemm_run", mtk.GroupedGemmArgs), ("mtk_grouped_grad_run", mtk.GroupedGradArgs), ("mtk_mx_quantize_run", mtk.MxQuantizeArgs),
            ("mtk_mx_dequantize_run", mtk.MxDequantizeArgs), ("mtk_mx_gemm_run", mtk.MxGemmArgs)]
    others = [p for p, _ in plans] + [mtk.GemmPlan(None, 64, 64, 64)]
    for i, (name, kind) in enumerate(runs):
        fn = getattr(L, name)
        assert fn(None, ctypes.byref(kind())) == INVALID
        for j, o in enumerate(others):
            if i != j:
                assert fn(o.handle, ctypes.byref(kind())) == INVALID and L.mtk_last_error()
    assert L.mtk_gemm_run(others[0].handle, ctypes.byref(mtk.GemmArgs())) == INVALID


@pytest.mark.parametrize("R, K", [(1, 1), (7, 255), (7, 256), (7, 257), (1000, 4100), (1 << 20, 1 << 14)])
def test_mx_bytes(R, K):
    k_tiles = -(-K // 256)
    assert mtk.mx_bytes(R, K) == (R * k_tiles * 128, R * k_tiles * 8)


def test_workspaces():
    # a plan needs one only where rows are brought into 4 bits by a launch of their own
    assert product().workspace_bytes == gradient(has_bias=True).workspace_bytes == quantise().workspace_bytes == few_bits().workspace_bytes == 0
    one = few_bits(T=1, N=4096, K=2048, quantize_a=True)
    assert one.workspace_bytes == 0 and one.describe().endswith("kernels: mtk_mx_gemm_f16_32q"), one.describe()
    many = few_bits(T=4000, N=4096, K=2000, quantize_a=True)
    codes, scales = mtk.mx_bytes(4000, 2000)
    assert codes + scales <= many.workspace_bytes < codes + scales + 256


# ------------------------------------------------------------------ the runtime, in C++

DRIVER = r"""
#include "runtime.cpp"
#include <new>
#include <random>
#include <set>

static int allocations = -1;  // that succeed before one fails; below 0: all
void *operator new(size_t n) {
  if (allocations == 0) throw std::bad_alloc();
  if (allocations > 0) --allocations;
  if (void *p = malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

static int failures = 0;
#define CHECK(x, ...) do { if (!(x)) { printf("failed: %s: ", #x); printf(__VA_ARGS__); printf("\n"); if (++failures > 20) exit(1); } } while (0)
static std::mt19937 rng(7);
static int upto(int n) { return (int)(rng() % (unsigned)n); }
static int about(int most) { return 1 + (int)std::exp(std::log((double)most) * (rng() % 10000) / 10000); }

// ---- groups, whatever row_start holds
static void groups() {
  const int odd[] = {0, 1, -1, 5, 99, 100, 101, INT32_MAX, INT32_MIN, INT32_MIN + 1, 64, 63};
  for (int a : odd)
    for (int b : odd) {
      const group_rows g = group_of(a, b, 100);
      CHECK(g.first >= 0 && g.rows >= 0 && g.first + g.rows <= 100, "%d %d: %d %d", a, b, g.first, g.rows);
      if (a >= 0 && a <= b && b <= 100) CHECK(g.first == a && g.rows == b - a, "%d %d", a, b);
      if (b <= a) CHECK(g.rows == 0, "%d %d", a, b);
    }
  for (int n = 0; n < 20000; ++n) {  // blocks of ascending groups, against the bound that a grid has
    const int E = 1 + upto(40), T = 1 + upto(2000), block = 32 << upto(4);
    std::vector<int> cut(E + 1);
    for (int &c : cut) c = upto(T + 1);
    std::sort(cut.begin(), cut.end());
    if (n % 2) cut[0] = 0, cut[E] = T;
    int64_t blocks = 0;
    for (int e = 0; e < E; ++e) blocks += (group_of(cut[e], cut[e + 1], T).rows + block - 1) / block;
    CHECK(blocks <= group_max_blocks(E, T, block), "E %d T %d block %d: %d", E, T, block, (int)blocks);
  }
}

// ---- every tile once, or its two halves once each, by one workgroup, and every workgroup comes to an end
static void tiles() {
  for (int n = 0; n < 20000; ++n) {
    const int total = upto(n % 3 ? 40 : 3000), grid = 1 + upto(n % 2 ? 600 : std::max(total, 1)), halves = upto(2);
    std::vector<int> had(2 * total, 0);
    int rounds = 0;
    for (int b = 0; b < grid; ++b)
      for (int i = 0;; ++i) {
        const group_place p = group_nth_tile(b, grid, i, total, halves);
        if (p.tile < 0) {
          CHECK(group_nth_tile(b, grid, i + 1, total, halves).tile < 0, "none, and one behind it");
          break;
        }
        CHECK(p.tile < total && p.half >= 0 && p.half <= 2 * halves, "tile %d of %d, half %d", p.tile, total, p.half);
        if (p.half != 2) ++had[2 * p.tile];
        if (p.half != 1) ++had[2 * p.tile + 1];
        rounds = std::max(rounds, i + 1);
      }
    for (int t = 0; t < 2 * total; ++t) CHECK(had[t] == 1, "half %d of %d, grid %d: %d times", t, 2 * total, grid, had[t]);
    CHECK(rounds == (total + grid - 1) / grid, "%d rounds", rounds);
  }
  for (int full = 0; full < 70; ++full)  // K-tiles from elsewhere on: each once, those behind the whole ones in their places
    for (int b = 0; b < 16; ++b) {
      const int turn = group_turn(b, full);
      CHECK(turn >= 0 && (turn < full || full == 0), "%d of %d", turn, full);
      std::set<int> seen;
      for (int k = 0; k < full; ++k) seen.insert(group_turned(k, turn, full));
      CHECK((int)seen.size() == full && (full == 0 || (*seen.begin() == 0 && *seen.rbegin() == full - 1)), "%d of %d", turn, full);
      CHECK(group_turned(full, turn, full) == full && group_turned(full + 1, turn, full) == full + 1, "%d", full);
    }
  for (int b = 0; b < 256; ++b) {  // no count passes 32 bits
    CHECK(group_nth_tile(b, 256, INT32_MAX / 256 - 1, INT32_MAX, 1).tile >= 0, " ");
    CHECK(group_nth_tile(b, 256, INT32_MAX / 256 + 1, INT32_MAX, 1).tile == -1, " ");
  }
}

// ---- rows that overlap, against every pair of them
static void rows() {
  int there = 0, apart = 0;
  char *const at = (char *)0x100000000ull;
  for (int n = 0; n < 40000; ++n) {
    const Rows a{"a", at, 1ull + rng() % 10, 2ull * (1 + rng() % 20), 0}, b{"b", at + 2 * (upto(300) - 150), 1ull + rng() % 10, 2ull * (1 + rng() % 20), 0};
    Rows x = a, y = b;
    x.step = std::max(a.width, b.width) + 2 * (rng() % 20);
    y.step = n % 3 ? x.step : b.width + 2 * (rng() % 20);
    bool want = false;
    for (uint64_t i = 0; i < x.n; ++i)
      for (uint64_t j = 0; j < y.n; ++j) want = want || overlap((const char *)x.at + i * x.step, x.width, (const char *)y.at + j * y.step, y.width);
    const bool got = meet(x, y);
    CHECK(got == meet(y, x), "both ways");
    // never missed; refused without need only between rows of different strides
    CHECK(want ? got : (!got || x.step != y.step || x.n < 2 || y.n < 2), "%d rows of %d, %d apart", (int)x.n, (int)x.width, (int)x.step);
    ++(want ? there : apart);
  }
  CHECK(there > 5000 && apart > 5000, "%d %d", there, apart);
}

// ---- each output against everything else that a run is given
static char *area(int i) { return (char *)0x100000000ull + ((size_t)i << 28); }
struct Field { const char *name; const void **at; size_t bytes; bool out; unsigned align; };
static void overlaps_of(const mtk_plan *p, const void *args, std::vector<Field> f) {
  CHECK(check_grouped_args(p, args) == MTK_OK, "%s", mtk_last_error());
  for (const Field &o : f) {
    if (!o.out) continue;
    for (const Field &x : f) {
      if (x.at == o.at) continue;
      const void *const keep = *x.at;
      auto put = [&](const char *to, bool refused) {
        *x.at = to;
        const int s = check_grouped_args(p, args);
        const bool said = s == MTK_ERR_INVALID && strstr(mtk_last_error(), "overlap") && strstr(mtk_last_error(), o.name) && strstr(mtk_last_error(), x.name);
        CHECK(refused ? said : s == MTK_OK, "%s and %s: %s", o.name, x.name, mtk_last_error());
      };
      auto up = [&](size_t n) { return (n + x.align - 1) / x.align * x.align; };
      const char *const at = (const char *)*o.at;
      put(at + (o.bytes - 1) / x.align * x.align, true);
      put(at + up(o.bytes), false);
      put(at - (x.bytes - 1) / x.align * x.align, true);
      put(at - up(x.bytes), false);
      *x.at = keep;
    }
    const void *const keep = *o.at;  // null
    *o.at = nullptr;
    CHECK(check_grouped_args(p, args) == MTK_ERR_INVALID, "%s null", o.name);
    if (o.align > 1) {
      *o.at = (const char *)keep + 1;
      CHECK(check_grouped_args(p, args) == MTK_ERR_INVALID && strstr(mtk_last_error(), "aligned"), "%s odd", o.name);
    }
    *o.at = keep;
  }
  for (const Field &x : f) {
    const void *const keep = *x.at;
    *x.at = nullptr;
    CHECK(check_grouped_args(p, args) == MTK_ERR_INVALID, "%s null", x.name);
    *x.at = (const char *)keep + x.align / 2;
    if (x.align > 1) CHECK(check_grouped_args(p, args) == MTK_ERR_INVALID && strstr(mtk_last_error(), "aligned"), "%s", x.name);
    *x.at = keep;
  }
  CHECK(check_grouped_args(p, nullptr) == MTK_ERR_INVALID, " ");
}
#define AT(x) (const void **)&x
static void arguments() {
  for (int odd = 0; odd < 2; ++odd)
    for (int t = 0; t < 2; ++t) {
      mtk_grouped_desc d{};
      d.E = 3, d.T = 50, d.N = 64, d.K = 96 + odd, d.trans_b = t, d.dtype = t, d.has_bias = 1;
      mtk_plan *p = nullptr, *g = nullptr;
      if (mtk_grouped_gemm_plan(nullptr, &d, &p)) exit(2);
      mtk_grouped_gemm_args a{area(0), area(1), area(2), (int32_t *)area(3), area(4), nullptr};
      const size_t x = 2 * d.T * d.K, y = 2 * d.T * d.N, w = 2 * d.E * d.N * d.K, b = 2 * d.E * d.N, r = 4 * (d.E + 1);
      const unsigned al = odd ? 2 : 4;
      overlaps_of(p, &a, {{"A", AT(a.A), x, false, al}, {"B", AT(a.B), w, false, odd && !t ? 2u : al}, {"bias", AT(a.bias), b, false, 2},
                          {"row_start", AT(a.row_start), r, false, 4}, {"C", AT(a.C), y, true, 2}});
      d.out_f32 = odd;
      if (mtk_grouped_grad_plan(nullptr, &d, &g)) exit(2);
      mtk_grouped_grad_args e{area(0), area(1), (int32_t *)area(2), area(3), area(4), nullptr};
      overlaps_of(g, &e, {{"A", AT(e.A), x, false, al}, {"dC", AT(e.dC), y, false, al}, {"row_start", AT(e.row_start), r, false, 4},
                          {"dB", AT(e.dB), w << odd, true, 16}, {"dbias", AT(e.dbias), b << odd, true, 4}});
      mtk_plan_destroy(p), mtk_plan_destroy(g);
    }
  mtk_mx_rows_desc d{50, 300, 0, MTK_BF16};
  mtk_plan *q = nullptr, *r = nullptr;
  if (mtk_mx_quantize_plan(nullptr, &d, &q) || mtk_mx_dequantize_plan(nullptr, &d, &r)) exit(2);
  const size_t codes = mx_code_bytes(50, 2), scales = mx_scale_bytes(50, 2);
  mtk_mx_quantize_args qa{area(0), area(1), area(2)};
  overlaps_of(q, &qa, {{"src", AT(qa.src), 2 * 50 * 300, false, 2}, {"codes", AT(qa.codes), codes, true, 16}, {"scales", AT(qa.scales), scales, true, 16}});
  mtk_mx_dequantize_args ra{area(0), area(1), area(2)};
  overlaps_of(r, &ra, {{"codes", AT(ra.codes), codes, false, 16}, {"scales", AT(ra.scales), scales, false, 16}, {"dst", AT(ra.dst), 2 * 50 * 300, true, 2}});
  for (int E = 0; E < 4; E += 3)
    for (int quant = 0; quant < 2; ++quant) {
      mtk_mx_gemm_desc m{};
      m.E = E, m.T = 5000, m.N = 640, m.K = 300, m.dtype = MTK_F16, m.has_bias = 1, m.quantize_a = quant;
      const int rows = (E ? E : 1) * m.N;
      mtk_plan *p = nullptr;
      if (mtk_mx_gemm_plan(nullptr, &m, &p)) exit(2);
      CHECK((p->workspace > 0) == (quant > 0), " ");
      mtk_mx_gemm_args a{area(0), quant ? nullptr : area(1), area(2), area(3), area(4), E ? (int32_t *)area(5) : nullptr, area(6), quant ? area(7) : nullptr};
      std::vector<Field> f = {{"A", AT(a.A), quant ? 2 * 5000 * 300 : mx_code_bytes(5000, 2), false, quant ? 2u : 16u}, {"B", AT(a.B), mx_code_bytes(rows, 2), false, 16},
                              {"b_scales", AT(a.b_scales), mx_scale_bytes(rows, 2), false, 16}, {"bias", AT(a.bias), 2 * (size_t)rows, false, 2},
                              {"C", AT(a.C), 2 * 5000 * 640, true, 2}};
      if (!quant) f.push_back({"a_scales", AT(a.a_scales), mx_scale_bytes(5000, 2), false, 16});
      if (E) f.push_back({"row_start", AT(a.row_start), 4 * (size_t)(E + 1), false, 4});
      if (quant) f.push_back({"workspace", AT(a.workspace), p->workspace, true, 16});
      overlaps_of(p, &a, f);
      // what a plan has no use for
      if (quant) {
        a.a_scales = area(1);
        CHECK(check_grouped_args(p, &a) == MTK_ERR_INVALID && strstr(mtk_last_error(), "a_scales"), " ");
        a.a_scales = nullptr;
      }
      if (!E) {
        a.row_start = (int32_t *)area(5);
        CHECK(check_grouped_args(p, &a) == MTK_ERR_INVALID && strstr(mtk_last_error(), "row_start"), " ");
      }
      mtk_plan_destroy(p);
    }
}

// ---- plans of every size: no count passes 32 bits, and the kernels that they choose
static std::set<std::string> names;
static bool take(mtk_plan *p) {
  if (!p) return false;
  for (const Launch &l : p->launches) {
    names.insert(l.name);
    CHECK(l.grid > 0 && (uint64_t)l.grid * l.block <= UINT32_MAX && l.block <= 1024, "%s: %u x %u", l.name.c_str(), l.grid, l.block);
  }
  mtk_plan_destroy(p);
  return true;
}
static void plans() {
  int made = 0;
  for (int n = 0; n < 60000; ++n) {
    const bool large = n % 4 == 0;
    const int E = large ? about(1 << 14) : about(200), T = large ? about(INT32_MAX - 8) : about(20000), N = about(large ? 1 << 22 : 16384), K = about(large ? 1 << 22 : 16384);
    const int pad = n % 3 ? 0 : 1 + upto(9);
    mtk_plan *p = nullptr;
    mtk_grouped_desc d{};
    d.E = E, d.T = T, d.N = N, d.K = n % 2 ? K : (K + 7) & ~7, d.trans_b = upto(2), d.dtype = upto(2), d.has_bias = upto(2);
    if (pad) d.lda = d.K + pad, d.ldc = d.N + pad;
    if (mtk_grouped_gemm_plan(nullptr, &d, &p) != MTK_OK) p = nullptr;
    made += take(p);
    d.out_f32 = upto(2);
    p = nullptr;
    if (mtk_grouped_grad_plan(nullptr, &d, &p) != MTK_OK) p = nullptr;
    made += take(p);
    mtk_mx_rows_desc r{T, K, pad ? K + pad : 0, upto(2)};
    p = nullptr;
    if ((n % 2 ? mtk_mx_quantize_plan : mtk_mx_dequantize_plan)(nullptr, &r, &p) != MTK_OK) p = nullptr;
    made += take(p);
    mtk_mx_gemm_desc m{};
    m.E = upto(2) ? E : 0, m.T = n % 5 ? T : about(64), m.N = N, m.K = K, m.dtype = upto(2), m.quantize_a = upto(2);
    p = nullptr;
    if (mtk_mx_gemm_plan(nullptr, &m, &p) != MTK_OK) p = nullptr;
    made += take(p);
  }
  CHECK(made > 100000, "%d plans", made);
}

// ---- every allocation of a plan's making fails once: an error, and no exception past the C entry
static void no_memory() {
  mtk_grouped_desc d{};
  d.E = 3, d.T = 50, d.N = 64, d.K = 96, d.has_bias = 1;
  mtk_mx_rows_desc r{50, 96, 0, MTK_F16};
  mtk_mx_gemm_desc m{};
  m.T = 5000, m.N = 640, m.K = 300, m.quantize_a = 1;
  for (int which = 0; which < 5; ++which) {
    int refused = 0;
    for (int n = 0;; ++n) {
      mtk_plan *p = nullptr;
      allocations = n;
      const int s = which == 0   ? mtk_grouped_gemm_plan(nullptr, &d, &p)
                    : which == 1 ? mtk_grouped_grad_plan(nullptr, &d, &p)
                    : which == 2 ? mtk_mx_quantize_plan(nullptr, &r, &p)
                    : which == 3 ? mtk_mx_dequantize_plan(nullptr, &r, &p)
                                 : mtk_mx_gemm_plan(nullptr, &m, &p);
      allocations = -1;
      if (s == MTK_OK) {
        mtk_plan_destroy(p);
        break;
      }
      CHECK(s == MTK_ERR_OOM && !p && strstr(mtk_last_error(), "memory"), "%d %d: %d", which, n, s);
      ++refused;
    }
    CHECK(refused >= 3, "%d: %d", which, refused);
  }
}

int main() {
  groups(), tiles(), no_memory(), rows(), arguments(), plans();
  for (const std::string &n : names) puts(n.c_str());
  return failures != 0;
}
"""


def test_runtime(tmp_path):
    scratch_obj = os.path.join(mtk.LIB_DIR, "scratch.o")
    if shutil.which("g++") is None or not os.path.exists(scratch_obj):
        pytest.skip("needs g++ and a built library (python -m example_matmul_metal4_amd.build)")
    src, exe = tmp_path / "grouped.cpp", tmp_path / "grouped"
    src.write_text(DRIVER)
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROCM}/include", f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), scratch_obj, f"-L{ROCM}/lib",
                        "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-ldl", "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    names = r.stdout.split()
    built = b"".join(open(f, "rb").read() for x in ("grouped", "mx") for f in glob.glob(os.path.join(mtk.LIB_DIR, f"mtk_{x}_*.hsaco")))
    have = {n.decode() for n in re.findall(rb"mtk_(?:grouped|mx)_[a-z0-9_]+(?=\.kd\0)", built)}
    assert have == set(names), have ^ set(names)  # none missing, and none that no plan runs


# ------------------------------------------------------------------ the numpy forms

def test_plain_product_and_its_gradients():
    # by loops over single elements, and the gradients against differences of the loss sum(C * dC)
    rng = np.random.default_rng(3)
    E, T, N, K = 3, 9, 4, 5
    starts = [2, 5, 5, 8]
    A, B, bias, dC = (kv.bits_of(rng.standard_normal(s), "bf16") for s in ((T, K), (E, N, K), (E, N), (T, N)))
    a, b, v, d = (kv.to_f64(x, "bf16") for x in (A, B, bias, dC))
    C, bound, mine = experts.grouped(A, B, bias, starts, True, "bf16")
    group = [-1, -1, 0, 0, 0, 2, 2, 2, -1]
    assert list(mine) == [g >= 0 for g in group]
    for t, e in enumerate(group):
        for n in range(N):
            want = sum(a[t, k] * b[e, n, k] for k in range(K)) + v[e, n] if e >= 0 else 0.0
            assert abs(C[t, n] - want) < 1e-12
    other, _, _ = experts.grouped(A, np.ascontiguousarray(B.transpose(0, 2, 1)), bias, starts, False, "bf16")
    assert np.abs(other - C).max() < 1e-12
    (dB, _), (dbias, _) = experts.grad(A, dC, starts, True, "bf16", "f32")
    (dBt, _), _ = experts.grad(A, dC, starts, False, "bf16", "f32")
    assert np.abs(dBt - dB.transpose(0, 2, 1)).max() < 1e-12 and (dB[1] == 0).all() and (dbias[1] == 0).all()

    def loss(b, v):
        return sum((d[t] * (b[e] @ a[t] + v[e])).sum() for t, e in enumerate(group) if e >= 0)

    for i in np.ndindex(E, N, K):
        step = np.zeros(b.shape)
        step[i] = 0.5  # the loss is linear: any step
        assert abs(loss(b + step, v) - loss(b - step, v) - dB[i]) < 1e-10
    for i in np.ndindex(E, N):
        step = np.zeros(v.shape)
        step[i] = 0.5
        assert abs(loss(b, v + step) - loss(b, v - step) - dbias[i]) < 1e-10
    # the input gradient is the forward product over the same weights, the other way round
    dA, _, _ = experts.grouped(dC, B, None, starts, False, "bf16")
    for t, e in enumerate(group):
        assert np.abs(dA[t] - (d[t] @ b[e] if e >= 0 else 0.0)).max() < 1e-12


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rows_in_4_bits(dtype):
    rng = np.random.default_rng(4)
    R, K = 5, 300
    x = kv.bits_of(rng.standard_normal((R, K)) * np.exp2(rng.integers(-10, 10, (R, 1))), dtype)
    x[1, 40] = kv.NAN_BITS[dtype]
    x[2, :32] = 0
    codes, scales = experts.quantise(x, dtype)
    assert codes.shape == (R, 256) and scales.shape == (2, R, 8)
    assert (codes.nbytes, scales.nbytes) == mtk.mx_bytes(R, K)
    v, f = experts.values(codes, scales, K), kv.to_f64(x, dtype)
    assert np.isnan(v[1, 32:64]).all() and np.isnan(v).sum() == 32
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    for r in range(R):
        for b in range(0, K, 32):
            blk = f[r, b:b + 32]
            if np.isnan(blk).any():
                continue
            s = 2.0 ** (int(scales[b // 256, r, b % 256 // 32]) - 127)
            most = np.abs(blk).max()
            assert most <= 6 * s and (most > 3 * s or s == 2.0 ** -126)
            near = np.abs(np.abs(blk)[:, None] / s - grid).min(1) * s  # to the nearest of the grid
            assert np.array_equal(np.abs(v[r, b:b + 32] - blk), near)
    assert (codes[:, 150:] == 0).all()  # places past K
