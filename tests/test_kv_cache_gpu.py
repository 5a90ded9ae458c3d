"""The paged key/value cache in few bits: rows written (bit for bit), read back (bit for bit) and attended to
(within a bound derived in oracle/kv.py), against numpy in 64 bits."""
import ctypes

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
import oracle
from oracle import kv

rng_of = lambda seed: np.random.default_rng(seed)


def rows16(rng, shape, dtype, size=1.0):
    return kv.bits_of(rng.standard_normal(shape) * size, dtype)


def table_of(rng, lens, page, spare=2, width=None):
    """(table, pages of the cache): every sequence's pages anywhere, entries past its length -1."""
    used = [-(-max(0, n) // page) for n in lens]
    n_pages = sum(used) + spare
    order = rng.permutation(n_pages)
    t = np.full((len(lens), width or max(1, max(used))), -1, np.int32)
    at = 0
    for b, n in enumerate(used):
        t[b, :n] = order[at:at + n]
        at += n
    return t, n_pages


def i32(x):
    return np.ascontiguousarray(x, np.int32)


class Batch:
    """A batch on the device and its cache on both sides."""

    def __init__(self, dev, seed, lens, rows, H_kv, D, page, fmt, dtype, fill=True, width=None):
        self.dev, rng = dev, rng_of(seed)
        self.lens, self.rows = i32(lens), list(rows)
        self.start = i32(np.concatenate([[0], np.cumsum(rows)]))
        self.table, n_pages = table_of(rng, lens, page, width=width)
        self.cache = kv.Cache(n_pages, page, H_kv, D, fmt, dtype)
        if fill:  # every byte of the pages: unused rows hold anything, NaN scales and codes among it
            self.cache.bytes[:] = rng.integers(0, 256, self.cache.bytes.size, dtype=np.uint8)
            for b, n in enumerate(lens):
                pos = np.arange(max(0, n))
                pages = self.cache.pages_of(self.table[b], pos)
                for p, o in zip(pages, pos % page):
                    for w in range(2):
                        self.cache.put(w, p, o, rows16(rng, (H_kv, D), dtype, 1.0 if w else 1.5))
        self.pages = dict(n_pages=n_pages, page_size=page, max_pages=self.table.shape[1], format=fmt, dtype=dtype)
        self.d = [dev.upload(x) for x in (self.cache.bytes, self.start, self.lens, self.table)]

    def free(self, *more):
        for x in self.d + list(more):
            x.free()

    def bytes_now(self):
        return self.dev.download(self.d[0], self.cache.bytes.shape, np.uint8)


def attend(batch, Q, H, causal=True, S_q=0, lse=True, fill=0x1234):
    dev, c = batch.dev, batch.cache
    T, D = Q.shape[0], c.D
    plan = mtk.KvAttentionPlan(dev, len(batch.lens), T, H, c.H_kv, D, S_q=S_q, causal=causal, **batch.pages)
    print(plan.describe(), flush=True)
    dq, do = dev.upload(Q), dev.upload(np.full(Q.shape, fill, np.uint16))
    dl = dev.upload(np.full((T, H), 77.0, np.float32)) if lse else None
    ws = dev.upload(np.full(plan.workspace_bytes, 0xFF, np.uint8)) if plan.workspace_bytes else None
    plan.run(dq, *batch.d, do, dl, ws)
    dev.sync()
    out = dev.download(do, Q.shape, np.uint16)
    ls = dev.download(dl, (T, H), np.float32) if lse else None
    for x in (dq, do, dl, ws):
        if x is not None:
            x.free()
    return out, ls


def check_attention(batch, Q, H, causal=True, S_q=0):
    got, lse = attend(batch, Q, H, causal, S_q)
    O, ref_lse, bound = batch.cache.attention(Q, batch.start, batch.lens, batch.table, causal, S_q)
    free = bound < 0  # rows that no sequence has
    assert (got[free] == 0x1234).all() and (lse[free[..., 0]] == 77.0).all()
    x = kv.to_f64(got, batch.cache.dtype)
    nan = np.isnan(O) & ~free
    assert np.array_equal(np.isnan(x) & ~free, nan)
    use = ~free & ~nan
    off = np.abs(x - O)[use]
    worst = (off / np.maximum(bound[use], 1e-300)).max() if off.size else 0.0
    print(f"worst {worst:.3f} of the bound", flush=True)
    assert (off <= bound[use]).all(), worst
    live = ~free[..., 0] & np.isfinite(ref_lse)
    assert np.array_equal(np.isneginf(lse)[~free[..., 0]], np.isneginf(ref_lse)[~free[..., 0]])
    # scores as in the bound above; the logarithm and its factor: a few steps of 32 bits
    assert (np.abs(lse - ref_lse)[live] <= 2e-5 * (1 + np.abs(ref_lse[live]))).all()
    dead = ~free[..., 0] & np.isnan(ref_lse)
    assert np.isnan(lse[dead]).all()
    return got


# ------------------------------------------------------------------ written and read back

HARD = ["normal", "any bits", "ties", "tiny", "huge", "zeros and NaN"]


def hard_rows(rng, shape, dtype, kind):
    if kind == "normal":
        return rows16(rng, shape, dtype)
    if kind == "any bits":  # most blocks hold a NaN or an infinity: one in four is kept finite
        x = rng.integers(0, 65536, shape).astype(np.uint16)
        keep = rng.random(shape[:-1] + (1,)) < 0.75
        return np.where(keep & ~np.isfinite(kv.to_f64(x, dtype)), x & 0x3FFF, x).astype(np.uint16)
    if kind == "ties":  # halves and quarters of powers of two: values between two codes
        return kv.bits_of(rng.integers(-64, 65, shape) / 2.0 ** rng.integers(0, 5, shape), dtype)
    if kind == "tiny":  # subnormals, and blocks whose scale is at its least
        return (rng.integers(0, 200, shape) | (rng.integers(0, 2, shape) << 15)).astype(np.uint16)
    if kind == "huge":
        most = 0x7BFF if dtype == "f16" else 0x7F7F
        return ((most - rng.integers(0, 600, shape)) | (rng.integers(0, 2, shape) << 15)).astype(np.uint16)
    x = np.zeros(shape, np.uint16)
    x[rng.random(shape) < 0.01] = kv.NAN_BITS[dtype]
    x[rng.random(shape) < 0.01] = 0x7C00 if dtype == "f16" else 0x7F80
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", HARD)
def test_rows_written_and_read_back(dev, fmt, dtype, kind):
    seed = 100 + HARD.index(kind)
    # (H_kv, D, page): a last block half empty, one block, 8-dim heads, many blocks
    for n, (H_kv, D, page) in enumerate([(2, 80, 16), (3, 32, 64), (1, 8, 16), (2, 256, 32)]):
        rng = rng_of(seed + n)
        b = Batch(dev, seed + n, [37, 5, 0, 64], [37, 3, 0, 1], H_kv, D, page, fmt, dtype)
        T = int(b.start[-1]) + 2  # two rows behind the last sequence
        K, V = (hard_rows(rng, (T, H_kv, D), dtype, kind) for _ in range(2))
        dK, dV = dev.upload(K), dev.upload(V)
        w = mtk.KvWritePlan(dev, 4, T, H_kv, D, **b.pages)
        w.run(dK, dV, *b.d)
        dev.sync()
        b.cache.write(K, V, b.start, b.lens, b.table)
        got = b.bytes_now()
        assert np.array_equal(got, b.cache.bytes), (H_kv, D, page, int((got != b.cache.bytes).sum()))
        r = mtk.KvReadPlan(dev, 4, T, H_kv, D, **b.pages)
        out = [dev.upload(np.full(K.shape, 0x1234, np.uint16)) for _ in range(2)]
        r.run(*b.d, *out)
        dev.sync()
        for x, want in zip(out, b.cache.read(T, b.start, b.lens, b.table, 0x1234)):
            x = dev.download(x, K.shape, np.uint16)
            nan = np.isnan(kv.to_f64(want, dtype))
            assert np.array_equal(np.isnan(kv.to_f64(x, dtype)), nan)
            bad = (x != want) & ~nan
            assert not bad.any(), (H_kv, D, page, x[bad][:5], want[bad][:5])
        b.free(dK, dV, *out)


@pytest.mark.gpu
def test_rows_of_a_fused_projection(dev):
    # K, V and Q as slices of one buffer [T][H + 2 H_kv][D]; what lies between the rows read back stays
    H, H_kv, D, page = 4, 2, 40, 16
    b = Batch(dev, 7, [50, 20], [9, 20], H_kv, D, page, "fp4", "bf16")
    T, ld = 29, (H + 2 * H_kv) * D
    qkv = rows16(rng_of(8), (T, H + 2 * H_kv, D), "bf16")
    d = dev.upload(qkv)
    at = lambda buf, heads: buf.ptr + 2 * heads * D
    mtk.KvWritePlan(dev, 2, T, H_kv, D, ld_k=ld, ld_v=ld, **b.pages).run(at(d, H), at(d, H + H_kv), *b.d)
    b.cache.write(qkv[:, H:H + H_kv], qkv[:, H + H_kv:], b.start, b.lens, b.table)
    dev.sync()
    assert np.array_equal(b.bytes_now(), b.cache.bytes)
    back = dev.upload(np.full(qkv.shape, 0x1234, np.uint16))
    mtk.KvReadPlan(dev, 2, T, H_kv, D, ld_k=ld, ld_v=ld, **b.pages).run(*b.d, at(back, H), at(back, H + H_kv))
    dev.sync()
    got = dev.download(back, qkv.shape, np.uint16)
    K, V = b.cache.read(T, b.start, b.lens, b.table, 0)
    assert (got[:, :H] == 0x1234).all() and np.array_equal(got[:, H:H + H_kv], K) and np.array_equal(got[:, H + H_kv:], V)
    plan = mtk.KvAttentionPlan(dev, 2, T, H, H_kv, D, ld_q=ld, **b.pages)
    o, ws = dev.empty(T * H * D * 2), dev.empty(max(1, plan.workspace_bytes))
    plan.run(d, *b.d, o, None, ws if plan.workspace_bytes else None)
    dev.sync()
    O, _, bound = b.cache.attention(np.ascontiguousarray(qkv[:, :H]), b.start, b.lens, b.table)
    assert (np.abs(kv.to_f64(dev.download(o, (T, H, D), np.uint16), "bf16") - O) <= bound).all()
    b.free(d, back, o, ws)


# ------------------------------------------------------------------ attention

# (lens, rows, H, H_kv, D, page, fmt, dtype, causal): one key; tiles of 32 keys and pages of 16 that end anywhere;
# sequences of no rows and of no positions; 1 to 300 (row, head) pairs per K/V head; every padded head dimension and
# blocks that are half empty; keys split over workgroups
CASES = [
    ([1], [1], 1, 1, 64, 16, "fp4", "f16", True),
    ([1, 2, 33], [1, 1, 1], 8, 2, 128, 16, "fp4", "bf16", True),
    ([15, 16, 17, 31, 32], [1] * 5, 4, 4, 40, 16, "fp4", "f16", True),
    ([127, 128, 129], [1] * 3, 8, 1, 128, 32, "fp8", "bf16", True),
    ([100, 0, 64], [3, 0, 64], 6, 2, 72, 16, "fp4", "f16", True),
    ([300, 77], [5, 5], 8, 2, 128, 64, "fp4", "bf16", True),
    ([90, 200], [7, 1], 14, 2, 256, 16, "fp4", "f16", True),
    ([200, 33], [2, 1], 6, 3, 200, 32, "fp8", "bf16", True),
    ([260], [100], 3, 1, 64, 64, "fp4", "bf16", True),
    ([140, 64], [40, 64], 4, 2, 96, 16, "fp8", "f16", False),
    ([500, 3], [9, 3], 8, 8, 128, 128, "fp4", "f16", False),
    ([3000], [1], 8, 2, 128, 16, "fp4", "bf16", True),
    ([4001, 100, 1500], [1, 1, 1], 4, 1, 64, 64, "fp8", "f16", True),
    ([2049, 700], [5, 2], 8, 2, 160, 256, "fp4", "bf16", True),
    ([1700], [30], 4, 1, 128, 32, "fp4", "f16", True),
    ([1030, 60], [300, 1], 2, 1, 128, 16, "fp4", "bf16", True),
    ([64, 64], [1, 1], 1, 1, 8, 1024, "fp4", "f16", True),
    ([600], [1], 71, 1, 64, 16, "fp4", "bf16", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(dev, case):
    lens, rows, H, H_kv, D, page, fmt, dtype, causal = case
    b = Batch(dev, 20, lens, rows, H_kv, D, page, fmt, dtype)
    T = int(b.start[-1]) + 1  # a row behind the last sequence
    Q = rows16(rng_of(21), (T, H, D), dtype)
    got = check_attention(b, Q, H, causal, S_q=max(rows))
    assert np.array_equal(got, attend(b, Q, H, causal, S_q=max(rows))[0])  # the same bits again
    b.free()
