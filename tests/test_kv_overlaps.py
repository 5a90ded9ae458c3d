"""Pointers of the paged cache's operators that overlap: what an operator writes meets neither what it reads, the batch's arrays
among it, nor its other outputs. Slices of one buffer, whose rows lie between each other, do not overlap. On the host."""
import os
import shutil
import subprocess

import pytest

import example_matmul_metal4_amd as mtk

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

PROGRAM = r"""
#include "runtime.cpp"
#include <random>

static int failures = 0;
#define CHECK(x, ...) do { if (!(x)) { printf("failed: %s: ", #x); printf(__VA_ARGS__); printf("\n"); if (++failures > 20) exit(1); } } while (0)

int main() {
  mtk_kv_desc d{};
  d.B = 3, d.T = 40, d.H = 8, d.H_kv = 2, d.D = 64, d.n_pages = 20, d.page_size = 16, d.max_pages = 600, d.dtype = MTK_F16;
  mtk_plan *w = nullptr, *r = nullptr, *t = nullptr;
  if (mtk_kv_write_plan(nullptr, &d, &w) || mtk_kv_read_plan(nullptr, &d, &r) || mtk_kv_attn_plan(nullptr, &d, &t)) return puts(mtk_last_error()), 1;
  char *const at = (char *)0x100000000ull;
  auto area = [&](int i) { return at + ((size_t)i << 28); };  // each operand in its own
  auto fine = [&](const mtk_plan *p, const void *x, const char *what) { CHECK(check_kv_args(p, x) == MTK_OK, "%s: %s", what, mtk_last_error()); };
  auto refused = [&](const mtk_plan *p, const void *x, const char *a, const char *b) {
    const bool is = check_kv_args(p, x) == MTK_ERR_INVALID && strstr(mtk_last_error(), a) && strstr(mtk_last_error(), b) &&
                    strstr(mtk_last_error(), "overlap");
    CHECK(is, "%s, %s: %s", a, b, mtk_last_error());
  };
  const char *const names[3] = {"row_start", "kv_len", "table"};
  const size_t sizes[3] = {4 * 4, 4 * 3, 4 * 3 * 600};
  const size_t cache = kv_cache_size(d), rows = 2 * 40 * 2 * 64, q = 2 * 40 * 8 * 64, lse = 4 * 40 * 8;

  // ---- each output against each array: the last bytes of one, and the first of the other
  mtk_kv_attn_args ta{area(0), area(1), (int32_t *)area(2), (int32_t *)area(3), (int32_t *)area(4), area(5), (float *)area(6), area(7)};
  fine(t, &ta, "attention");
  CHECK(t->workspace > 0, " ");
  void **const outs[3] = {&ta.O, (void **)&ta.lse, &ta.workspace};
  const char *const out_names[3] = {"O", "lse", "workspace"};
  const size_t out_sizes[3] = {q, lse, t->workspace};
  for (int o = 0; o < 3; ++o)
    for (int i = 0; i < 3; ++i) {
      const mtk_kv_attn_args keep = ta;
      const int32_t **x = &ta.row_start + i;
      *x = (const int32_t *)((char *)*outs[o] + out_sizes[o] - 4);
      refused(t, &ta, out_names[o], names[i]);
      *x = (const int32_t *)((char *)*outs[o] + (out_sizes[o] + 3) / 4 * 4);
      fine(t, &ta, "behind an output");
      *x = (const int32_t *)((char *)*outs[o] - sizes[i] + 4);
      refused(t, &ta, out_names[o], names[i]);
      *x = (const int32_t *)((char *)*outs[o] - sizes[i]);
      fine(t, &ta, "before an output");
      ta = keep;
    }
  ta.lse = (float *)((char *)ta.O + q - 4);
  refused(t, &ta, "lse", "O");

  mtk_kv_write_args wa{area(0), area(1), area(2), (int32_t *)area(3), (int32_t *)area(4), (int32_t *)area(5)};
  fine(w, &wa, "write");
  mtk_kv_read_args ra{area(2), (int32_t *)area(3), (int32_t *)area(4), (int32_t *)area(5), area(0), area(1)};
  fine(r, &ra, "read");
  for (int i = 0; i < 3; ++i) {
    mtk_kv_write_args x = wa;
    (&x.row_start)[i] = (const int32_t *)((char *)wa.cache + cache - 4);
    refused(w, &x, "cache", names[i]);
    (&x.row_start)[i] = (const int32_t *)wa.K;  // read only, both of them
    fine(w, &x, "arrays and K");
    for (int v = 0; v < 2; ++v) {
      mtk_kv_read_args y = ra;
      (&y.row_start)[i] = (const int32_t *)((char *)(v ? ra.V : ra.K) + rows - 4);
      refused(r, &y, v ? "V" : "K", names[i]);
      (&y.row_start)[i] = (const int32_t *)ra.cache;
      fine(r, &y, "arrays and the cache");
    }
  }

  // ---- rows of K and V read back: parts of each other, slices of one buffer
  mtk_kv_read_args x = ra;
  x.V = (char *)ra.K + rows - 16;
  refused(r, &x, "K", "V");
  x.V = (char *)ra.K - rows + 16;
  refused(r, &x, "K", "V");
  x.V = (char *)ra.K + rows;
  fine(r, &x, "V behind K");
  x.V = (char *)ra.K - rows;
  fine(r, &x, "V before K");
  std::mt19937 rng(3);
  int meet = 0, apart = 0;
  for (int n = 0; n < 20000; ++n) {  // against every pair of rows
    const int T = 1 + rng() % 12, width = 8 * (1 + rng() % 6);
    const int64_t ld_a = width + 8 * (rng() % 20), ld_b = rng() % 2 ? ld_a : width + 8 * (rng() % 20);
    const char *a = at, *b = at + 16 * ((int)(rng() % 400) - 200);
    bool want = false;
    for (int i = 0; i < T; ++i)
      for (int j = 0; j < T; ++j) want = want || overlap(a + 2 * i * ld_a, 2 * width, b + 2 * j * ld_b, 2 * width);
    CHECK(rows_meet(a, ld_a, b, ld_b, T, width) == want, "T %d width %d strides %d %d apart %d", T, width, (int)ld_a, (int)ld_b, (int)(b - a));
    ++(want ? meet : apart);
  }
  CHECK(meet > 3000 && apart > 3000, "%d %d", meet, apart);
  return failures != 0;
}
"""


def test_overlaps(tmp_path):
    scratch_obj = os.path.join(mtk.LIB_DIR, "scratch.o")
    if shutil.which("g++") is None or not os.path.exists(scratch_obj):
        pytest.skip("needs g++ and a built library (python -m example_matmul_metal4_amd.build)")
    src, exe = tmp_path / "overlaps.cpp", tmp_path / "overlaps"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROCM}/include", f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), scratch_obj, f"-L{ROCM}/lib",
                        "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-ldl", "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
