"""Attention over the paged cache for batches whose sequences may all have many rows and long tables: that they are planned,
and who does what then (every step of every pair once, sums that fit 32 bits), whatever the arrays on the device hold."""
import os
import shutil
import subprocess

import pytest

import example_matmul_metal4_amd as mtk

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def plan(B, T, S_q, H, H_kv, D, positions, page=16, **kw):
    return mtk.KvAttentionPlan(None, B, T, H, H_kv, D, S_q=S_q, n_pages=100, page_size=page, max_pages=positions // page, **kw)


@pytest.mark.parametrize("B, T, S_q, H, H_kv, D, positions", [
    (256, 4351, 4096, 32, 8, 128, 131072),   # a chunk of up to 4096 rows beside 255 tokens
    (256, 8447, 0, 32, 8, 128, 131072),
    (64, 4159, 4096, 64, 8, 128, 1 << 20),   # a context of a million positions
    (1024, 17000, 16000, 64, 8, 128, 131072),
    (512, 2048, 2048, 16, 16, 256, 1 << 20),
    (300, 2000, 2000, 8, 2, 64, 1 << 27),
])
def test_batches_are_planned(B, T, S_q, H, H_kv, D, positions):
    d = plan(B, T, S_q, H, H_kv, D, positions).describe()
    assert "mtk_kv_attend" in d and "mtk_kv_prefill" in d
    # the grid covers the packed rows, not S_q of every sequence
    grid = int(d.split("rows/wg=128 grid=")[1].split()[0])
    assert grid <= max(512, H_kv * (T * (H // H_kv) // 128 + B))


def test_batches_past_the_sums_are_refused():
    for kw in (dict(B=40000, T=100000, S_q=100000, H=128, H_kv=64, D=64, positions=1024),  # 2^29 blocks of 128 rows
               dict(B=1 << 20, T=1 << 20, S_q=256, H=16, H_kv=16, D=64, positions=1024)):  # more workgroups than a grid has
        with pytest.raises(mtk.MtkError) as e:
            plan(**kw)
        assert e.value.status == mtk.MTK_ERR_UNSUPPORTED and e.value.message


PROGRAM = r"""
#include "runtime.cpp"
#include <random>

static int failures = 0;
#define CHECK(x, ...) do { if (!(x)) { printf("failed: %s: ", #x); printf(__VA_ARGS__); printf("\n"); if (++failures > 20) exit(1); } } while (0)

int main() {
  std::mt19937 rng(12);
  auto log = [&](int64_t lo, int64_t hi) { return (int64_t)(lo * std::pow((double)hi / lo, std::uniform_real_distribution<>(0, 1)(rng))); };
  int longer = 0, shared = 0;
  for (int n = 0; n < 6000; ++n) {
    mtk_kv_desc d{};
    const int groups[] = {1, 2, 4, 8};
    d.B = (int)log(1, 600), d.H_kv = 1 << rng() % 5, d.H = d.H_kv * groups[rng() % 4], d.D = 64 << rng() % 3, d.T = (int)log(100, 20000);
    d.S_q = rng() % 2 ? 0 : (int)log(50, d.T + 1), d.page_size = 16 << rng() % 7, d.max_pages = (int)(log(1 << 12, 1 << 24) / d.page_size);
    d.n_pages = 1000, d.format = rng() % 2, d.dtype = rng() % 2, d.causal = 1;
    if (d.S_q > d.T) d.S_q = d.T;
    if (d.max_pages < 1) d.max_pages = 1;
    mtk_plan *p = nullptr;
    if (mtk_kv_attn_plan(nullptr, &d, &p) != MTK_OK) {
      CHECK(0, "%s", mtk_last_error());
      continue;
    }
    for (Launch &l : p->launches) {
      if (l.name.find("prefill") == std::string::npos) continue;
      const mtk_kv_prefill_kargs &both = args_of<mtk_kv_prefill_kargs>(l);
      const mtk_kv_attn_kargs &k = both.rows;
      const int64_t grid = l.grid - both.joins, cap = (int64_t)d.max_pages * d.page_size;
      longer += k.step_shift > 6;
      CHECK(k.step_shift >= 6 && k.least >= 1 && ((int64_t)k.least << k.step_shift) >= std::min<int64_t>(cap, 256), "shift %d least %d", k.step_shift, k.least);
      for (int kind = 0; kind < 4; ++kind) {  // ragged; one chunk beside tokens; every table full; starts that do not ascend
        std::vector<int> start(d.B + 1), len(d.B);
        for (int b = 0; b <= d.B; ++b) start[b] = kind == 3 ? (int)rng() : (int)(rng() % (d.T + 1));
        if (kind != 3) std::sort(start.begin(), start.end());
        if (kind == 1) for (int b = 0; b <= d.B; ++b) start[b] = b < d.B ? std::min(b, d.T) : d.T;
        for (int b = 0; b < d.B; ++b) len[b] = kind >= 2 ? INT32_MAX : (int)log(1, cap + 1);
        if (kind == 3) for (int b = 0; b <= d.B; ++b) start[b] = b % 2 ? INT32_MAX : -1;  // every other one claims all the rows
        int64_t work = 0, own = 0;
        std::vector<kv_share> h;
        for (int b = 0; b < d.B; ++b) {
          const kv_seq s = kv_sequence(start[b], start[b + 1], len[b], k.T, k.max_pages, k.page_shift);
          h.push_back(kv_blocks(s, k.S_q, k.G, k.rows_shift, k.step_shift, k.rows_above, k.rows_most));
          work += (int64_t)h[b].blocks * k.H_kv * h[b].steps;
          own += (int64_t)h[b].blocks * k.H_kv;
        }
        CHECK(work <= INT32_MAX && own <= INT32_MAX, "work %lld own %lld", (long long)work, (long long)own);
        const int most = (int)((cap + ((int64_t)1 << k.step_shift) - 1) >> k.step_shift), few = kv_few_steps(k.step_shift);
        kv_cut cut = {kv_each_of_pairs((int)work, (int)own, k.units, k.least, most, few), 1};
        CHECK(cut.each >= 1, "each %d", cut.each);
        int64_t line = 0, wgs = 0;
        for (auto &x : h) {
          const int64_t pairs = (int64_t)x.blocks * k.H_kv;
          const int length = kv_length(x, cut);
          CHECK(length >= x.steps && length % cut.each == 0, "length %d of %d", length, x.steps);
          line += pairs * length, wgs += pairs * (length / cut.each);
          if (length > cut.each) ++shared;
          if (length > cut.each) CHECK(k.places > 0, "shared without room: %s", p->description.c_str());
        }
        CHECK(line + cut.each <= INT32_MAX, "line %lld each %d: %s", (long long)line, cut.each, p->description.c_str());
        if (kind == 3) continue;  // rows claimed twice
        CHECK(wgs <= grid, "%lld workgroups of %lld: %s", (long long)wgs, (long long)grid, p->description.c_str());
        if (kv_pairs_split((int)work, (int)own, k.units, few)) CHECK(wgs <= k.units, "%lld workgroups", (long long)wgs);
      }
    }
    mtk_plan_destroy(p);
  }
  if (longer < 500 || shared < 1000) return printf("%d with longer steps, %d shared\n", longer, shared), 1;
  return failures != 0;
}
"""


def test_schedule(tmp_path):
    scratch_obj = os.path.join(mtk.LIB_DIR, "scratch.o")
    if shutil.which("g++") is None or not os.path.exists(scratch_obj):
        pytest.skip("needs g++ and a built library (python -m example_matmul_metal4_amd.build)")
    src, exe = tmp_path / "large.cpp", tmp_path / "large"
    src.write_text(PROGRAM)
    r = subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROCM}/include", f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), scratch_obj, f"-L{ROCM}/lib",
                        "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-ldl", "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
