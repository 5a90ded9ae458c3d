"""A row of a grouped product has the same bits whatever rows the other groups have and wherever its own group starts: results of a
serving batch do not depend on who else is in it. On every kernel whose tiles go through K from different places."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

FILL = 0x1234
EQUAL = 16  # the group's rows repeat after so many

# operator, kernel, E, T, N, K, dtype, 16-bit rows
CASES = [
    ("grouped", "nt_256", 10, 1976, 3250, 1104, "bf16", True), ("grouped", "nt_256", 11, 2494, 2574, 1080, "f16", True),
    ("grouped", "nt_128", 28, 80, 1223, 1056, "f16", True), ("grouped", "nt_128", 48, 1807, 640, 1100, "bf16", True),
    ("grouped", "nt_64_w8", 2, 60, 102, 2100, "bf16", True), ("grouped", "nt_64_w4", 51, 69, 408, 1088, "bf16", True),
    ("grouped", "nt_64_w1", 24, 60, 3092, 1054, "f16", True), ("grouped", "nt_64_any_w8", 2, 60, 123, 2101, "f16", True),
    ("grouped", "nt_64_any_w4", 59, 127, 257, 1121, "bf16", True), ("grouped", "nt_64_any_w1", 10, 21, 7537, 1189, "f16", True),
    ("mx", "256", 4, 1676, 5345, 2304, "f16", True), ("mx", "128", 48, 1807, 624, 2200, "f16", False),
    ("mx", "64", 34, 2459, 140, 2100, "bf16", False), ("mx", "32", 2, 60, 102, 4200, "bf16", False), ("mx", "32q", 2, 26, 125, 1120, "f16", True),
]


def plan_of(dev, op, E, T, N, K, dtype, rows16):
    if op == "grouped":
        return mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype, has_bias=True)
    return mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, has_bias=True, quantize_a=rows16)


def routings(E, T, rows):
    """Some row_start in which group E // 2 has `rows` rows, other rows lie before it and behind it, and the rows of the others vary."""
    g, rest = E // 2, T - rows
    for before in sorted({0, 1, min(37, rest // 2), rest // 2, rest - 1, rest}):
        for groups in (1, g):  # in one group before it, or spread over all of them
            starts = np.zeros(E + 1, int)
            starts[g - groups:g + 1] = np.linspace(0, before, groups + 1).round()
            starts[g + 1:] = np.linspace(before + rows, T, E - g).round() if E - g > 1 else T
            starts[g + 1] = before + rows
            yield starts.astype(np.int32)


def test_the_kernels_are_those():
    for op, kernel, *rest in CASES:
        assert plan_of(None, op, *rest).describe().split("16_")[-1] == kernel, (op, kernel)


def cancelling(rng, E, N, K, dtype):
    """EQUAL rows and the weights of E groups, of places of very different sizes, whose second half takes the sum of the first one away again:
    what is left are the roundings on the way (and the few places behind), so that another order of the additions shows in the result's
    bits."""
    X, W = rng.standard_normal((EQUAL, K)), rng.standard_normal((E, N, K))
    half = K // 512 * 256
    size = np.exp2(rng.integers(0, 11, half // 32)).repeat(32)
    X[:, :half] *= size
    W[:, :, :half] *= size
    X[:, half:2 * half] = -X[:, :half]
    W[:, :, half:2 * half] = W[:, :, :half]
    return kv.bits_of(X, dtype), kv.bits_of(W.reshape(E * N, K), dtype)


PLACES = r"""
#include "groups.h"
#include <cstdio>
#include <initializer_list>
int main() {
  for (int log_parts = 0; log_parts < 4; ++log_parts)
    for (int across : {1, 2, 3, 5, 7, 8, 9, 31, 32, 33, 100, 224, 1000, 4097, 40000, 65535, 65536}) {
      const group_turns t = group_turns_of(log_parts, across);
      const int step = 8 >> log_parts;
      int last = -1, parts = 0;
      for (int n = 0; n < across; ++n) {  // parts of neighbouring columns, in order, each about as wide as the others
        const int p = group_turn_place(0, n, t);
        if (!t.on || p % step || p < 0 || p >= 8 || p < last) return printf("%d of %d, %d parts: %d\n", n, across, 1 << log_parts, p), 1;
        parts += p != last;
        last = p;
        if (group_turn_place(16383, n, t) - p != group_turn_place(16383, 0, t)) return 2;
      }
      if (across >= 1 << log_parts ? parts != 1 << log_parts : parts != across) return printf("%d: %d parts\n", across, parts), 3;
    }
  int had = 0;
  for (int e = 0; e < 8; ++e) had |= 1 << (group_turn_place(e, 0, group_turns_of(0, 1)) & 7);
  if (had != 255) return 4;  // eight groups in a row start at eight places
  for (int e = 0; e < 64; ++e)
    if (!((group_turn_place(e, 0, group_turns_of(0, 1)) - group_turn_place(e + 8, 0, group_turns_of(0, 1))) & 7)) return 5;
  return 0;
}
"""


def test_places(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    src, exe = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PLACES)
    subprocess.run(["g++", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{os.path.join(mtk.PKG, 'csrc')}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[6]}")
def test_bits_of_a_row(dev, case):
    op, kernel, E, T, N, K, dtype, rows16 = case
    rng = np.random.default_rng(K + T)
    rows, g = max(1, T // 3), E // 2
    X, W = cancelling(rng, E, N, K, dtype)
    X = X[np.arange(rows) % EQUAL]
    A, bias = kv.bits_of(rng.standard_normal((T, K)), dtype), kv.bits_of(np.zeros((E, N)), dtype)
    plan = plan_of(dev, op, E, T, N, K, dtype, rows16)
    print(plan.describe(), flush=True)
    weights = [dev.upload(x) for x in ([W] if op == "grouped" else experts.quantise(W, dtype))]
    d_bias, C, ws = dev.upload(bias), dev.empty(2 * T * N), dev.empty(max(16, plan.workspace_bytes))
    first = None
    for starts in routings(E, T, rows):
        at = starts[g]
        assert starts[g + 1] - at == rows and (np.diff(starts) >= 0).all() and starts[-1] <= T
        batch = A.copy()
        batch[at:at + rows] = X
        ds = dev.upload(starts)
        dev.upload_into(C, np.full((T, N), FILL, np.uint16))
        if op == "grouped":
            a = [dev.upload(batch)]
            plan.run(a[0], weights[0], d_bias, ds, C)
        else:
            a = [dev.upload(x) for x in ([batch] if rows16 else experts.quantise(batch, dtype))]
            plan.run(a[0], None if rows16 else a[1], *weights, d_bias, ds, C, ws)
        dev.sync()
        got = dev.download(C, (T, N), np.uint16)[at:at + rows]
        for x in (*a, ds):
            x.free()
        if first is None:
            first = got
            assert (got != 0).any()
        off = np.argwhere(got != first)
        assert len(off) == 0, f"{len(off)} of {got.size} values of the same rows differ, the first at {off[:3].tolist()}, behind {at} other rows"
        off = np.argwhere(got != got[np.arange(rows) % EQUAL])
        assert len(off) == 0, f"{len(off)} of {got.size} values of equal rows of the group differ, the first at {off[:3].tolist()}"
    for x in (*weights, d_bias, C, ws):
        x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("op, E, T, N, K, dtype, rows16", [
    ("grouped", 1, 1000, 700, 1100, "bf16", True), ("grouped", 1, 1900, 6000, 1100, "f16", True), ("grouped", 1, 300, 333, 1101, "f16", True),
    ("mx", 0, 150, 700, 4200, "bf16", True), ("mx", 0, 1000, 2000, 2100, "f16", False), ("mx", 0, 1900, 9000, 2304, "bf16", True), ("mx", 1, 900, 640, 2304, "f16", False),
], ids=str)
def test_bits_of_equal_rows_of_one_group(dev, op, E, T, N, K, dtype, rows16):
    rng = np.random.default_rng(K + T)
    X, W = cancelling(rng, 1, N, K, dtype)
    A = X[np.arange(T) % EQUAL]
    plan = plan_of(dev, op, E, T, N, K, dtype, rows16)
    print(plan.describe(), flush=True)
    d = [dev.upload(x) for x in ([W] if op == "grouped" else experts.quantise(W, dtype))]
    a = [dev.upload(x) for x in ([A] if rows16 else experts.quantise(A, dtype))]
    bias, C, ws = dev.upload(np.zeros(N, np.uint16)), dev.empty(2 * T * N), dev.empty(max(16, plan.workspace_bytes))
    got = []
    for first in (0, 1, 5) if E else (0,):
        starts = dev.upload(np.array([first, T], np.int32)) if E else None
        if op == "grouped":
            plan.run(a[0], d[0], bias, starts, C)
        else:
            plan.run(a[0], None if rows16 else a[1], *d, bias, starts, C, ws)
        dev.sync()
        out = dev.download(C, (T, N), np.uint16)[first:]
        got.append(out[(np.arange(T - first) + first) % EQUAL == 0])
        assert (out == out[(np.arange(T - first)) % EQUAL]).all(), f"equal rows differ behind {first} rows of no group"
        if starts is not None:
            starts.free()
    assert all((g == got[0][0]).all() for g in got)
    for x in (*d, *a, bias, C, ws):
        x.free()
