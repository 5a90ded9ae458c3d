"""Sizes that plans of grouped and 4-bit products take, and where they end: as include/mtk.h states it, on both sides of each border.
Those near a launch's limits run on the GPU."""
import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

UNSUPPORTED = mtk.MTK_ERR_UNSUPPORTED
FILL = 0x1234


def forward(E, T, N, K, **kw):
    return mtk.GroupedGemmPlan(None, E, T, N, K, **kw)


def gradient(E, T, N, K, **kw):
    return mtk.GroupedGradPlan(None, E, T, N, K, **kw)


def kernels(plan):
    return plan.describe().split("kernels: ")[1].split()


def refused(make, *a, **kw):
    with pytest.raises(mtk.MtkError) as e:
        make(*a, **kw)
    return e.value.status == UNSUPPORTED and e.value.message


@pytest.mark.parametrize("make, size", [
    (forward, (1, 1 << 20, 32767, 1)), (forward, (1, 1 << 18, 151936, 511)), (gradient, (512, 16, 32767, 1023)),  # odd: tiles of 64
    (forward, (1 << 14, 1 << 16, 14336, 64)),  # more tiles of 64 than 32 bits count, if row_start held every row in every group
    (forward, (1, 1 << 30, 64, 96)), (forward, (1, 1 << 30, 1, 1)), (forward, (4, 1 << 22, 1 << 14, 64)), (gradient, (64, 100, 1 << 16, 1 << 16)),
], ids=str)
def test_large_plans(make, size):
    for dtype in ("f16", "bf16"):
        for bias in (False, True):
            assert kernels(make(*size, dtype=dtype, has_bias=bias))


def up(n, d):
    return -(-n // d)


@pytest.mark.parametrize("odd", [0, 1])
def test_borders_of_forward_products(odd):
    # T up to 2^30
    assert kernels(forward(2, 1 << 30, 64, 2 + odd, lda=2 + odd)) and refused(forward, 2, (1 << 30) + 1, 64, 2 + odd)
    # E x ceil(T / t) x ceil(N / t) below 2^31, t 64 where a leading dimension is odd, else 256
    t = 64 if odd else 256
    E, N = 1 << 14, 1 << 12
    T = t * ((1 << 31) // E // (N // t))
    assert refused(forward, E, T, N, 2 + odd) and kernels(forward(E, T - t, N, 2 + odd))
    # (floor(T / 64) + E) x ceil(N / 64) below 2^26 where it is odd, the count of one launch
    E, T, N = 2, 1 << 20, (1 << 18) - 1
    assert (T // 64 + E) * up(N, 64) >= 1 << 26 > (T // 64 + E) * (up(N, 64) - 1)
    if odd:
        assert refused(forward, E, T, N, 3) and kernels(forward(E, T, N - 64, 3))
    else:
        assert kernels(forward(E, T, N, 2))


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("bias", [False, True])
def test_borders_of_gradients(odd, bias):
    E, T, N = 1 << 14, 4, 100
    K = (1 << 22) - 1 if not odd else 64 * ((1 << 26) // E // 2) - 1
    if not odd:
        assert kernels(gradient(E, T, N, K - 1, has_bias=bias))
        return
    # E x (ceil(N / 64) x ceil(K / 64) + ceil(N / 64)), the latter with a bias, below 2^26
    tiles = E * (up(N, 64) * up(K, 64) + (up(N, 64) if bias else 0))
    assert tiles >= 1 << 26 and refused(gradient, E, T, N, K, has_bias=bias)
    less = K - 64 * (2 if bias else 1)
    assert kernels(gradient(E, T, N, less, has_bias=bias))


@pytest.mark.parametrize("K", [1, 256, 257, 2048, 1 << 22])
def test_borders_of_4_bits(K):
    # rows x ceil(K / 256) up to 2^28 - 32, of A and of B, and what a product takes can be brought into the format and back
    rows = ((1 << 28) - 32) // up(K, 256)
    for quantize_a in (False, True):
        assert kernels(mtk.MxGemmPlan(None, rows, 1, K, quantize_a=quantize_a))
        message = refused(mtk.MxGemmPlan, None, rows + 1, 1, K, quantize_a=quantize_a)
        assert "2^28 - 32" in message
    E = up(rows, 1 << 22)
    N = rows // E
    assert kernels(mtk.MxGemmPlan(None, 1, N, K, E=E))
    assert refused(mtk.MxGemmPlan, None, 1, N + 1 + 32 // E, K, E=E) or N == 1 << 22
    for make in (mtk.MxQuantizePlan, mtk.MxDequantizePlan):
        assert kernels(make(None, rows, K))
        # ceil(R / 16) x ceil(K / 512) below 2^24
        most = 16 * (((1 << 24) - 1) // up(K, 512))
        assert kernels(make(None, most, K)) and refused(make, None, most + 1, K)


@pytest.mark.gpu
def test_rows_of_many_small_tiles(dev):
    # 2^22 tiles and more, of one row block and column each
    E, T, N, K, dtype = 2, (1 << 28) + 323, 1, 1, "bf16"
    rng = np.random.default_rng(1)
    values = kv.bits_of(np.array([1.0, -1.5, 2.0, 0.0, -0.25]), dtype)
    A, B = values[rng.integers(0, 5, T, dtype=np.uint8)], kv.bits_of(np.array([2.0, -0.5]), dtype)
    cut = 200_000_001
    plan = mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype)
    print(plan.describe(), flush=True)
    d = [dev.upload(A), dev.upload(B), None, dev.upload(np.array([3, cut, T], np.int32)), dev.empty(2 * (T + 64))]
    dev.fill_u16(d[4], FILL, T + 64)
    plan.run(*d)
    dev.sync()
    C = dev.download(d[4], (T + 64,), np.uint16)
    assert (C[:3] == FILL).all() and (C[T:] == FILL).all()
    for b, (i, j) in zip((2.0, -0.5), ((3, cut), (cut, T))):
        for v in values:
            want = kv.bits_of(kv.to_f64(v[None], dtype) * b, dtype)[0]
            got = C[i:j][A[i:j] == v]
            assert ((got == want) | ((got | want) & 0x7FFF == 0)).all(), (b, v)  # zeros of either sign
    for x in d:
        if x is not None:
            x.free()


@pytest.mark.gpu
def test_gradients_of_many_small_tiles(dev):
    # 2^25 tiles and more, a wavefront each: more than 2^31 threads
    E, T, N, K, dtype = 1 << 14, 5, 1, 131_201, "bf16"
    rng = np.random.default_rng(2)
    A, dC = kv.bits_of(rng.integers(-4, 5, (T, K)), dtype), kv.bits_of(rng.integers(-4, 5, (T, N)), dtype)
    starts = np.zeros(E + 1, np.int32)
    starts[8000:], starts[E - 1:] = 2, 4
    starts[E] = T
    plan = mtk.GroupedGradPlan(dev, E, T, N, K, dtype=dtype)
    print(plan.describe(), flush=True)
    n = E * N * K
    d = [dev.upload(A), dev.upload(dC), dev.upload(starts), dev.empty(2 * (n + 64))]
    dev.fill_u16(d[3], FILL, n + 64)
    plan.run(*d)
    dev.sync()
    got = dev.download(d[3], (n + 64,), np.uint16)
    assert (got[n:] == FILL).all()
    got = got[:n].reshape(E, K)
    a, g = kv.to_f64(A, dtype), kv.to_f64(dC, dtype)[:, 0]
    want = np.zeros((E, K))
    rest = np.ones(E, bool)
    for e, (i, j) in ((7999, (0, 2)), (E - 2, (2, 4)), (E - 1, (4, 5))):
        want = (g[i:j, None] * a[i:j]).sum(0)  # small whole numbers: exact
        assert np.array_equal(kv.to_f64(got[e], dtype), want), e
        rest[e] = False
    assert not got[rest].any()
    for x in d:
        x.free()


@pytest.mark.gpu
def test_rows_into_4_bits_of_many_workgroups(dev):
    # more than 2^23 workgroups, 2^31 threads: one value a row, of those that a block of one value holds exactly
    R, K, dtype = (1 << 27) + 77, 1, "bf16"
    rng = np.random.default_rng(3)
    values = kv.bits_of(np.array([0.0, 1.0, -1.5, 2.0, -3.0, 2.0 ** -120, 1.5 * 2.0 ** 100]), dtype)
    x = values[rng.integers(0, len(values), R, dtype=np.uint8)]
    src, back = dev.upload(x), dev.empty(2 * (R + 64))
    codes, scales = (dev.empty(n) for n in mtk.mx_bytes(R, K))  # 17 GB and 1 GB
    dev.fill_u16(back, FILL, R + 64)
    there, here = mtk.MxQuantizePlan(dev, R, K, dtype=dtype), mtk.MxDequantizePlan(dev, R, K, dtype=dtype)
    print(there.describe(), here.describe(), flush=True)
    there.run(src, codes, scales)
    here.run(codes, scales, back)
    dev.sync()
    got = dev.download(back, (R + 64,), np.uint16)
    assert (got[R:] == FILL).all() and np.array_equal(got[:R], x)
    # the last rows' codes, padding and all
    row = codes.nbytes // R
    last = dev.download(mtk.DeviceBuffer(dev, codes.ptr + (R - 9) * row, 9 * row), (9, row), np.uint8)
    assert np.array_equal(last, experts.quantise(x[R - 9:, None], dtype)[0])
    for b in (src, back, codes, scales):
        b.free()
