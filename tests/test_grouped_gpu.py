"""Products grouped by expert (forward, input gradient, gradients of weights and bias) against numpy in 64 bits, within a bound
derived in oracle/experts.py. What no group has, what lies between rows and what lies behind the outputs stays as it was."""
import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

rng_of = lambda seed: np.random.default_rng(seed)
i32 = lambda x: np.ascontiguousarray(x, np.int32)
FILL = 0x1234


def rows16(rng, shape, dtype, size=1.0):
    return kv.bits_of(rng.standard_normal(shape) * size, dtype)


def starts_of(rng, T, E, how):
    """row_start [E + 1]: random, one group with all, groups of one row, a hole before the first and behind the last."""
    if how == "one":
        e = int(rng.integers(0, E))
        return i32([0] * (e + 1) + [T] * (E - e))
    if how == "hole":
        cuts = np.sort(rng.integers(min(3, T), max(min(3, T) + 1, T - 5), E + 1))
        return i32(cuts)
    if how == "even":
        return i32(np.linspace(0, T, E + 1).round())
    cuts = np.sort(rng.integers(0, T + 1, E - 1))
    return i32(np.concatenate([[0], cuts, [T]]))


def strided(x, ld, fill):
    """[n][width] in rows of ld elements, filled between them, and a guard row behind the last."""
    out = np.full((x.shape[0] + 1, ld), fill, np.uint16)
    out[:-1, :x.shape[1]] = x
    return out


def check(got, want, bound, what):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])


def run_grouped(dev, A, B, bias, starts, trans_b, dtype, pad=(0, 0, 0), plan=None, repeat=True):
    """C's rows [T][N] after the product, over rows of FILL; pad: what the leading dimensions have more than the rows. repeat:
    the same bits again (not of rows that two groups claim, which either of them may write last)."""
    T, K = A.shape
    E, N = B.shape[0], B.shape[1] if trans_b else B.shape[2]
    lda, ldb, ldc = K + pad[0], B.shape[2] + pad[1], N + pad[2]
    plan = plan or mtk.GroupedGemmPlan(dev, E, T, N, K, trans_b=trans_b, dtype=dtype, has_bias=bias is not None,
                                       lda=lda, ldb=ldb, ldc=ldc)
    print(plan.describe(), flush=True)
    nan = kv.NAN_BITS[dtype]  # between the rows: never to be used
    da = dev.upload(strided(A, lda, nan)[:-1])
    db = dev.upload(strided(B.reshape(-1, B.shape[2]), ldb, nan)[:-1])
    dbias = dev.upload(bias) if bias is not None else None
    ds, dc = dev.upload(i32(starts)), dev.upload(np.full((T + 1, ldc), FILL, np.uint16))
    ws = dev.upload(np.full(plan.workspace_bytes, 0xFF, np.uint8)) if plan.workspace_bytes else None
    plan.run(da, db, dbias, ds, dc, ws)
    dev.sync()
    out = dev.download(dc, (T + 1, ldc), np.uint16)
    if repeat:
        plan.run(da, db, dbias, ds, dc, ws)
        dev.sync()
        assert np.array_equal(out, dev.download(dc, (T + 1, ldc), np.uint16))
    for x in (da, db, dbias, ds, dc, ws):
        if x is not None:
            x.free()
    assert (out[:, N:] == FILL).all() and (out[T] == FILL).all()
    return out[:T, :N]


def check_grouped(dev, A, B, bias, starts, trans_b, dtype, pad=(0, 0, 0)):
    out = run_grouped(dev, A, B, bias, starts, trans_b, dtype, pad)
    want, bound, mine = experts.grouped(A, B, bias, starts, trans_b, dtype)
    assert (out[~mine] == FILL).all()
    check(kv.to_f64(out, dtype)[mine], want[mine], bound[mine], "C")
    return out


# E, T, N, K, trans_b, dtype, bias, how, pad
CASES = [
    (1, 1, 1, 1, True, "f16", True, "even", (0, 0, 0)),
    (4, 1, 64, 64, True, "bf16", False, "random", (0, 0, 0)),
    (5, 3, 65, 130, True, "f16", True, "random", (0, 0, 0)),
    (5, 3, 66, 130, False, "bf16", True, "random", (0, 0, 0)),
    (3, 200, 100, 200, True, "bf16", False, "random", (8, 8, 8)),
    (3, 200, 100, 200, False, "f16", True, "hole", (8, 8, 8)),
    (7, 150, 101, 77, True, "f16", True, "random", (0, 0, 0)),
    (7, 150, 101, 77, False, "bf16", False, "hole", (0, 0, 0)),
    (7, 150, 90, 77, False, "f16", False, "random", (1, 3, 5)),
    (2, 90, 96, 300, True, "bf16", True, "one", (1, 0, 1)),
    (100, 130, 48, 64, True, "f16", True, "random", (0, 0, 0)),
    (200, 130, 48, 72, False, "bf16", False, "hole", (0, 0, 0)),
    (66, 700, 200, 520, True, "bf16", True, "random", (0, 0, 0)),
    (2, 17, 512, 1024, True, "f16", True, "random", (0, 0, 0)),
    # 128 x 128 tiles
    (3, 300, 10240, 136, True, "f16", True, "random", (0, 0, 0)),
    (3, 300, 10240, 136, False, "bf16", False, "random", (0, 0, 0)),
    (5, 500, 5000, 100, True, "bf16", False, "hole", (2, 4, 6)),
    # 256 x 256 tiles
    (3, 700, 12800, 136, True, "bf16", True, "random", (0, 0, 0)),
    (3, 700, 12800, 100, False, "f16", True, "hole", (0, 0, 0)),
    (6, 1500, 6000, 70, True, "f16", False, "random", (4, 2, 0)),
    (70, 6000, 2000, 64, False, "bf16", False, "random", (0, 0, 0)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_grouped_product(dev, case):
    E, T, N, K, trans_b, dtype, with_bias, how, pad = case
    rng = rng_of(100 + E + T)
    A, B = rows16(rng, (T, K), dtype), rows16(rng, (E, N, K) if trans_b else (E, K, N), dtype, 1 / np.sqrt(K))
    bias = rows16(rng, (E, N), dtype) if with_bias else None
    check_grouped(dev, A, B, bias, starts_of(rng, T, E, how), trans_b, dtype, pad)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,trans_b", [(40, 70, 100, True), (40, 70, 101, False), (400, 12800, 72, True), (400, 12800, 72, False)])
def test_rows_depend_on_their_own_group_only(dev, T, N, K, trans_b):
    """NaN and infinities in one group's rows, another's weights, and rows of no group reach no other row."""
    rng, dtype, E = rng_of(7), "bf16", 5
    A, B = rows16(rng, (T, K), dtype), rows16(rng, (E, N, K) if trans_b else (E, K, N), dtype)
    c = T // 8
    starts = i32([c, 3 * c, 3 * c, 5 * c - 1, 6 * c, 7 * c])
    clean = run_grouped(dev, A, B, None, starts, trans_b, dtype)
    A2, B2 = A.copy(), B.copy()
    A2[:c], A2[7 * c:] = 0x7FC0, 0x7F80  # no group's
    A2[3 * c:5 * c - 1:2] = 0x7FC0  # every other row of group 2
    B2[1], B2[3] = 0x7FC0, 0x7F80  # the group without rows, and group 3
    out = run_grouped(dev, A2, B2, None, starts, trans_b, dtype)
    keep = np.ones(T, bool)
    keep[3 * c:5 * c - 1:2] = False
    keep[5 * c - 1:6 * c] = False
    assert np.array_equal(out[keep], clean[keep])
    assert np.isnan(kv.to_f64(out[3 * c:5 * c - 1:2], dtype)).all()
    assert not np.isfinite(kv.to_f64(out[5 * c - 1:6 * c], dtype)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [64, 12800])
def test_row_starts_out_of_range(dev, N):
    """Whatever row_start holds, nothing but C's rows is written; ascending entries out of [0, T] are limited to it."""
    rng, dtype, T, K, E = rng_of(8), "f16", 400, 64, 4
    A, B = rows16(rng, (T, K), dtype), rows16(rng, (E, N, K), dtype)
    check_grouped(dev, A, B, None, i32([-5, 17, 17, 300, 2 ** 31 - 1]), True, dtype)
    check_grouped(dev, A, B, None, i32([-2 ** 31, -7, 0, 0, 0]), True, dtype)
    check_grouped(dev, A, B, None, i32([T, T + 1, T + 2, T + 3, T + 9]), True, dtype)
    run_grouped(dev, A, B, None, i32([0, T, 0, T, 0]), True, dtype, repeat=False)
    run_grouped(dev, A, B, None, i32([300, 200, 100, 50, 2]), True, dtype)


# E, T, N, K, trans_b, dtype, bias, out_f32, how, pad
GRADS = [
    (1, 1, 1, 1, True, "f16", True, False, "even", (0, 0)),
    (4, 1, 64, 64, True, "bf16", True, True, "random", (0, 0)),
    (5, 30, 65, 130, True, "f16", True, True, "random", (0, 0)),
    (5, 30, 66, 130, False, "bf16", True, False, "random", (0, 0)),
    (3, 200, 100, 201, True, "bf16", True, True, "hole", (8, 8)),
    (3, 200, 100, 200, False, "f16", True, False, "random", (2, 4)),
    (7, 150, 101, 77, False, "bf16", True, True, "random", (0, 0)),
    (7, 150, 101, 77, True, "f16", True, False, "one", (1, 2)),
    (90, 100, 40, 64, True, "bf16", True, True, "random", (0, 0)),
    (40, 500, 256, 256, True, "f16", True, True, "random", (0, 0)),
    (30, 300, 250, 300, False, "bf16", False, False, "hole", (0, 0)),
    (12, 600, 1024, 1020, True, "bf16", True, False, "random", (0, 0)),
    (12, 600, 1023, 1026, True, "f16", False, True, "random", (1, 0)),
    (20, 700, 1022, 777, False, "f16", False, True, "random", (0, 1)),
]


def run_grad(dev, A, dC, starts, trans_b, dtype, with_bias, out_f32, pad=(0, 0), plan=None):
    T, K, N, E = A.shape[0], A.shape[1], dC.shape[1], len(starts) - 1
    plan = plan or mtk.GroupedGradPlan(dev, E, T, N, K, trans_b=trans_b, dtype=dtype, has_bias=with_bias, out_f32=out_f32,
                                       lda=K + pad[0], ldc=N + pad[1])
    print(plan.describe(), flush=True)
    nan, kind = kv.NAN_BITS[dtype], np.float32 if out_f32 else np.uint16
    da, dd = dev.upload(strided(A, K + pad[0], nan)[:-1]), dev.upload(strided(dC, N + pad[1], nan)[:-1])
    ds = dev.upload(i32(starts))
    sizes = [E * N * K, E * N]
    outs = [dev.upload(np.full(n + 64, FILL, kind)) for n in sizes]
    ws = dev.upload(np.full(plan.workspace_bytes, 0xFF, np.uint8)) if plan.workspace_bytes else None
    got = []
    for _ in range(2):
        plan.run(da, dd, ds, outs[0], outs[1] if with_bias else None, ws)
        dev.sync()
        got.append([dev.download(o, (n + 64,), kind) for o, n in zip(outs, sizes)])
    for x, y, n in zip(got[0], got[1], sizes):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8)) and (x[n:] == FILL).all()
    if not with_bias:
        assert (got[0][1] == FILL).all()
    for x in [da, dd, ds, ws] + outs:
        if x is not None:
            x.free()
    return got[0][0][:sizes[0]].reshape((E, N, K) if trans_b else (E, K, N)), got[0][1][:sizes[1]].reshape(E, N)


def check_grad(dev, A, dC, starts, trans_b, dtype, with_bias, out_f32, pad=(0, 0)):
    dB, dbias = run_grad(dev, A, dC, starts, trans_b, dtype, with_bias, out_f32, pad)
    w, b = experts.grad(A, dC, starts, trans_b, dtype, "f32" if out_f32 else dtype)
    val = (lambda x: x.astype(np.float64)) if out_f32 else (lambda x: kv.to_f64(x, dtype))
    check(val(dB), *w, "dB")
    if with_bias:
        check(val(dbias), *b, "dbias")


@pytest.mark.gpu
@pytest.mark.parametrize("case", GRADS, ids=str)
def test_gradients(dev, case):
    E, T, N, K, trans_b, dtype, with_bias, out_f32, how, pad = case
    rng = rng_of(200 + E + T)
    A, dC = rows16(rng, (T, K), dtype), rows16(rng, (T, N), dtype)
    check_grad(dev, A, dC, starts_of(rng, T, E, how), trans_b, dtype, with_bias, out_f32, pad)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(72, 100), (71, 99), (1024, 1024)])
def test_gradients_of_groups_beside_nan(dev, N, K):
    """Rows of other groups and of none, NaN and infinities, reach no gradient but their own; no row: zeros."""
    rng, dtype, E, T = rng_of(9), "bf16", 12, 150
    A, dC = rows16(rng, (T, K), dtype), rows16(rng, (T, N), dtype)
    starts = i32([5, 5, 70, 71, 71, 71, 100, 110, 120, 130, 130, 131, 140])
    clean = run_grad(dev, A, dC, starts, True, dtype, True, True)
    for x in (A, dC):
        x[:5], x[140:], x[70] = 0x7FC0, 0x7F80, 0x7FC0
    dB, dbias = run_grad(dev, A, dC, starts, True, dtype, True, True)
    for e in range(E):
        if e == 2:
            assert np.isnan(dB[e]).all() and np.isnan(dbias[e]).all()
        else:
            assert np.array_equal(dB[e], clean[0][e]) and np.array_equal(dbias[e], clean[1][e])
    for e in (0, 3, 4, 9):
        assert not dB[e].any() and not dbias[e].any()


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """sum(C * G) with values of few bits, so that steps of a weight, an input and a bias change it exactly: the three gradients are
    its differences."""
    rng, E, T, N, K = rng_of(10), 3, 20, 24, 40
    A, B = rng.integers(-4, 5, (T, K)).astype(np.float64), rng.integers(-4, 5, (E, N, K)).astype(np.float64)
    bias, G = rng.integers(-4, 5, (E, N)).astype(np.float64), rng.integers(-2, 3, (T, N)).astype(np.float64)
    starts = i32([0, 7, 7, 20])
    h = lambda x: kv.bits_of(x, "f16")

    def loss(A, B, bias):
        out = run_grouped(dev, h(A), h(B), h(bias), starts, True, "f16")
        return float((kv.to_f64(out, "f16") * G).sum())

    dB, dbias = run_grad(dev, h(A), h(G), starts, True, "f16", True, True)
    dA = kv.to_f64(run_grouped(dev, h(G), h(B), None, starts, False, "f16"), "f16")  # the same weights, [E][N][K] as [E][K'][N']
    base = loss(A, B, bias)
    for x, g, at in ((B, dB, (0, 3, 5)), (B, dB, (2, 20, 39)), (B, dB, (1, 1, 1)), (bias, dbias, (0, 23)), (bias, dbias, (2, 0)),
                     (A, dA, (6, 39)), (A, dA, (7, 0))):
        y = x.copy()
        y[at] += 1
        new = loss(*(y if v is x else v for v in (A, B, bias)))
        assert new - base == g[at], (at, new - base, g[at])
