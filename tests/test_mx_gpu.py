"""Rows in blocks of 32 four-bit values (bit for bit) and products of them (within a bound derived in oracle/experts.py) against
numpy in 64 bits."""
import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

rng_of = lambda seed: np.random.default_rng(seed)
i32 = lambda x: np.ascontiguousarray(x, np.int32)
FILL = 0x1234


def activations(rng, shape, dtype):
    """Rows with a few large places, and blocks of every size."""
    x = rng.standard_normal(shape) * np.where(rng.random(shape[1:]) < 0.02, 20.0, 1.0)
    return kv.bits_of(x * 2.0 ** rng.integers(-6, 7, shape[:1] + (1,)), dtype)


def quantise(dev, x, dtype, ld=0):
    R, K = x.shape
    plan = mtk.MxQuantizePlan(dev, R, K, dtype=dtype, ld=ld)
    host = np.full((R, ld or K), kv.NAN_BITS[dtype], np.uint16)
    host[:, :K] = x
    nc, ns = mtk.mx_bytes(R, K)
    dx, dc, ds = dev.upload(host), dev.upload(np.full(nc + 32, 0xA5, np.uint8)), dev.upload(np.full(ns + 32, 0xA5, np.uint8))
    plan.run(dx, dc, ds)
    dev.sync()
    codes, scales = dev.download(dc, (nc + 32,), np.uint8), dev.download(ds, (ns + 32,), np.uint8)
    assert (codes[nc:] == 0xA5).all() and (scales[ns:] == 0xA5).all()
    for b in (dx, dc, ds):
        b.free()
    return codes[:nc].reshape(R, -1), scales[:ns].reshape(-1, R, 8)


def dequantise(dev, codes, scales, K, dtype, ld=0):
    R = codes.shape[0]
    plan = mtk.MxDequantizePlan(dev, R, K, dtype=dtype, ld=ld)
    dc, ds, dx = dev.upload(codes), dev.upload(scales), dev.upload(np.full((R + 1, ld or K), FILL, np.uint16))
    plan.run(dc, ds, dx)
    dev.sync()
    out = dev.download(dx, (R + 1, ld or K), np.uint16)
    assert (out[R] == FILL).all() and (out[:, K:] == FILL).all()
    for b in (dx, dc, ds):
        b.free()
    return out[:R, :K]


ROWS = [(1, 1, 0), (1, 32, 0), (3, 33, 0), (5, 256, 0), (4, 257, 264), (9, 511, 0), (2, 520, 523), (33, 1000, 1000), (70, 4100, 0),
        (1025, 300, 304), (6, 768, 1536), (2, 14336, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R,K,ld", ROWS)
def test_rows(dev, R, K, ld, dtype):
    x = activations(rng_of(R + K), (R, K), dtype)
    codes, scales = quantise(dev, x, dtype, ld)
    want = experts.quantise(x, dtype)
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])
    back = dequantise(dev, codes, scales, K, dtype, ld)
    assert np.array_equal(kv.to_f64(back, dtype), kv.to_f64(kv.bits_of(experts.values(*want, K), dtype), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_value(dev, dtype):
    """Every 16-bit pattern among moderate ones: subnormals, the largest, infinities and NaN; blocks of one size each."""
    bits = np.arange(65536, dtype=np.uint16)
    mixed = np.stack([bits, np.roll(bits, 7919)]).reshape(-1, 512)
    alone = np.where(np.arange(32) == 5, bits[:, None], 0).astype(np.uint16).reshape(-1, 1024)
    sorted_ = np.sort(bits.view(np.int16)).view(np.uint16).reshape(-1, 1024)
    for x in (mixed, alone, sorted_):
        codes, scales = quantise(dev, x, dtype)
        want = experts.quantise(x, dtype)
        bad = np.repeat(want[1] == 255, 16, -1).transpose(1, 0, 2).reshape(codes.shape)  # codes of a NaN block are of no matter
        assert np.array_equal(scales, want[1])
        assert np.array_equal(np.where(bad, 0, codes), np.where(bad, 0, want[0]))
        back = kv.to_f64(dequantise(dev, codes, scales, x.shape[1], dtype), dtype)
        v = kv.to_f64(kv.bits_of(experts.values(*want, x.shape[1]), dtype), dtype)
        assert np.array_equal(np.isnan(back), np.isnan(v)) and np.array_equal(back[~np.isnan(v)], v[~np.isnan(v)])
        assert not np.isinf(back).any()


def product(dev, A, B, bias, starts, dtype, quantize_a, ldc=0, lda=0, K=None):
    """A: 16-bit rows or (codes, scales); B: (codes, scales) of all rows."""
    T, E = (A if quantize_a else A[0]).shape[0], len(starts) - 1 if starts is not None else 0
    N = B[0].shape[0] // max(1, E)
    plan = mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, has_bias=bias is not None, quantize_a=quantize_a, ldc=ldc,
                          lda=lda if quantize_a else 0)
    print(plan.describe(), flush=True)
    host = None
    if quantize_a:
        host = np.full((T, lda or K), kv.NAN_BITS[dtype], np.uint16)
        host[:, :K] = A
    da, dsa = (dev.upload(host), None) if quantize_a else (dev.upload(A[0]), dev.upload(A[1]))
    db, dsb = dev.upload(B[0]), dev.upload(B[1])
    dbias = dev.upload(bias) if bias is not None else None
    ds = dev.upload(i32(starts)) if starts is not None else None
    dc = dev.upload(np.full((T + 1, ldc or N), FILL, np.uint16))
    ws = dev.upload(np.full(plan.workspace_bytes, 0xFF, np.uint8)) if plan.workspace_bytes else None
    outs = []
    for _ in range(2):
        plan.run(da, dsa, db, dsb, dbias, ds, dc, ws)
        dev.sync()
        outs.append(dev.download(dc, (T + 1, ldc or N), np.uint16))
    assert np.array_equal(outs[0], outs[1])  # the same bits again
    for b in (da, dsa, db, dsb, dbias, ds, dc, ws):
        if b is not None:
            b.free()
    assert (outs[0][T] == FILL).all() and (outs[0][:, N:] == FILL).all()
    return outs[0][:T, :N]


def check(got, want, bound):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])


# E, T, N, K, dtype, bias, quantize_a, ldc - N, lda - K
CASES = [
    (0, 1, 1, 1, "f16", True, True, 0, 0),
    (0, 1, 64, 256, "bf16", False, False, 0, 0),
    (0, 5, 70, 300, "f16", True, True, 3, 5),
    (0, 16, 512, 4096, "bf16", True, True, 0, 0),
    (0, 33, 1000, 520, "f16", False, True, 0, 8),
    (0, 130, 200, 4100, "bf16", True, True, 1, 0),
    (0, 64, 64, 2048, "f16", False, False, 0, 0),
    (0, 300, 700, 64, "bf16", False, True, 0, 0),
    (3, 40, 70, 300, "bf16", True, True, 0, 0),
    (5, 3, 65, 130, "f16", True, False, 0, 0),
    (70, 200, 96, 512, "bf16", False, True, 0, 0),
    (1, 90, 128, 256, "f16", True, True, 0, 0),
    (0, 600, 10240, 300, "f16", True, True, 0, 0),
    (3, 700, 12800, 136, "bf16", True, True, 0, 0),
    (70, 6000, 2000, 64, "f16", False, True, 0, 0),
    (0, 1100, 5000, 777, "bf16", True, False, 6, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_product(dev, case):
    E, T, N, K, dtype, with_bias, quantize_a, pad_c, pad_a = case
    rng, groups = rng_of(300 + T + N), max(1, E)
    A = activations(rng, (T, K), dtype)
    W = kv.bits_of(rng.standard_normal((groups * N, K)) / np.sqrt(K), dtype)
    bias = kv.bits_of(rng.standard_normal((groups, N)), dtype) if with_bias else None
    starts = None
    if E:
        starts = i32(np.concatenate([[min(1, T - 1)], np.sort(rng.integers(1, T, E - 1)), [T]]))
    qa, qb = experts.quantise(A, dtype), experts.quantise(W, dtype)
    out = product(dev, A if quantize_a else qa, qb, bias, starts, dtype, quantize_a, N + pad_c, K + pad_a, K)
    want, bound, mine = experts.mx_product(experts.values(*qa, K), experts.values(*qb, K).reshape(groups, N, K), bias,
                                           starts if E else [0, T], dtype)
    assert (out[~mine] == FILL).all()
    check(kv.to_f64(out, dtype)[mine], want[mine], bound[mine])


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(3, 70), (40, 70), (500, 10240)])
def test_nan_blocks_and_extreme_scales(dev, T, N):
    """A NaN block makes the outputs of its row (of A) and column (of B) NaN and no others; the smallest and the largest
    scales multiply as the numbers that they stand for."""
    K, dtype = 600, "bf16"
    rng = rng_of(11)
    A, W = activations(rng, (T, K), dtype), kv.bits_of(rng.standard_normal((N, K)), dtype)
    A[1, 300], W[66, 5], W[0, 599] = 0x7FC0, 0x7F80, 0xFF80
    A[0] = kv.bits_of(kv.to_f64(A[0], dtype) * 2.0 ** -100, dtype)
    W[3] = kv.bits_of(kv.to_f64(W[3], dtype) * 2.0 ** 100, dtype)
    A[2] = kv.bits_of(kv.to_f64(A[2], dtype) * 2.0 ** 110, dtype)
    W[4] = kv.bits_of(kv.to_f64(W[4], dtype) * 2.0 ** -100, dtype)
    qa, qb = experts.quantise(A, dtype), experts.quantise(W, dtype)
    out = kv.to_f64(product(dev, qa, qb, None, None, dtype, False, K=K), dtype)
    bad = np.zeros((T, N), bool)
    bad[1], bad[:, 66], bad[:, 0] = True, True, True
    assert np.isnan(out[bad]).all()
    with np.errstate(invalid="ignore"):
        want, bound, _ = experts.mx_product(experts.values(*qa, K), experts.values(*qb, K)[None], None, [0, T], dtype)
    # of row 2 and column 3 the largest are past the type: held out, as is what falls below the smallest normal number
    fits = ~bad & (np.abs(want) < 2.0 ** 126) & ((np.abs(want) > 2.0 ** -118) | (np.arange(T)[:, None] > 0))
    check(out[fits], want[fits], bound[fits])
