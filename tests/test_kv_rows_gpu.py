"""Rows written into the paged cache and read back by wavefronts that have several rows each, as prompts have them: sequences that
begin and end within a wavefront's rows, rows without a page or a sequence between them. Bit for bit against numpy."""
import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import kv
from test_kv_cache_gpu import hard_rows, i32, rng_of, rows16

pytestmark = pytest.mark.gpu


def places(cache, T, start, lens, table):
    """(sequence has it, page, offset) of each packed row."""
    has, page, off = np.zeros(T, bool), np.full(T, -1), np.zeros(T, np.int64)
    for b, first, n, pos0 in cache._rows(T, start, lens):
        pos = pos0 + np.arange(n)
        has[first:first + n] = True
        page[first:first + n] = cache.pages_of(table[b], pos)
        off[first:first + n] = pos % cache.page
    return has, page, off


def write(cache, K, V, page, off):
    """All rows at once; no two have the same place."""
    ok = page >= 0
    for w, x in enumerate((K, V)):
        codes, scales = kv.quantise(x[ok], cache.fmt, cache.dtype)
        flat = codes.reshape(codes.shape[0], cache.H_kv, -1)
        if cache.fmt == "fp4":
            flat = flat[..., 0::2] | (flat[..., 1::2] << 4)
        cache.part(w, False)[page[ok], :, off[ok]] = flat
        cache.part(w, True)[page[ok], :, off[ok]] = scales


# (K/V heads, dims, rows, rows of a wavefront): a head of 8 dims leaves most lanes without one; blocks that are half empty; several
# wavefronts to a row
SIZES = [(1, 8, 4101, 2), (1, 8, 8203, 4), (3, 80, 2049, 2), (3, 80, 4099, 4), (8, 128, 1031, 2), (8, 128, 2057, 4), (2, 256, 2050, 2)]


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("most", [7, 400])
@pytest.mark.parametrize("H_kv, D, T, per_wave", SIZES)
def test_several_rows_of_a_wavefront(dev, H_kv, D, T, per_wave, most, dtype, fmt):
    rng, page = rng_of(95 + most), 16
    rows, used = [], 0
    while used < T - 10:  # sequences of 0 to `most` rows, some rows in front and behind
        rows.append(min(int(rng.integers(0, most + 1)), T - 10 - used))
        used += rows[-1]
    B = len(rows)
    assert B > 64 or most > 7
    start = i32(np.concatenate([[0], np.cumsum(rows)])) + 5
    lens = i32(np.array(rows) + rng.integers(0, 40, B))
    lens[B // 3] = rows[B // 3] // 2  # its first rows lie before position 0
    need = [-(-int(n) // page) for n in lens]
    width, n_pages = max(need), sum(need) + 2
    order, table, at = rng.permutation(n_pages), np.full((B, width), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    gone = rng.random(table.shape) < 0.1  # pages that are none
    table = i32(np.where(gone, rng.choice([-1, n_pages, 1 << 30], table.shape), table))
    lens[B // 2] = width * page + rows[B // 2]  # rows past the table
    c = kv.Cache(n_pages, page, H_kv, D, fmt, dtype)
    c.bytes[:] = rng.integers(0, 256, c.bytes.size, dtype=np.uint8)
    pages = dict(n_pages=n_pages, page_size=page, max_pages=width, format=fmt, dtype=dtype)
    K, V = rows16(rng, (T, H_kv, D), dtype), hard_rows(rng, (T, H_kv, D), dtype, "any bits")
    has, at_page, at_off = places(c, T, start, lens, table)
    assert not has.all() and (has & (at_page < 0)).any() and (at_page >= 0).sum() > T / 8
    dK, dV, cache, *batch = [dev.upload(x) for x in (K, V, c.bytes, start, lens, table)]
    w = mtk.KvWritePlan(dev, B, T, H_kv, D, **pages)
    r = mtk.KvReadPlan(dev, B, T, H_kv, D, **pages)
    print(w.describe(), flush=True)
    assert f"rows/wave={per_wave} " in w.describe() and f"rows/wave={per_wave} " in r.describe()
    w.run(dK, dV, cache, *batch)
    dev.sync()
    write(c, K, V, at_page, at_off)
    got = dev.download(cache, c.bytes.shape, np.uint8)
    assert np.array_equal(got, c.bytes), int((got != c.bytes).sum())
    out = [dev.upload(np.full(K.shape, 0x1234, np.uint16)) for _ in range(2)]
    r.run(cache, *batch, *out)
    dev.sync()
    for which, x in enumerate(out):
        got = dev.download(x, K.shape, np.uint16)
        want = np.where(has[:, None, None], kv.bits_of(c.values(which, at_page, at_off), dtype), np.uint16(0x1234))
        nan = np.isnan(kv.to_f64(want, dtype))
        assert np.array_equal(np.isnan(kv.to_f64(got, dtype)), nan)
        assert np.array_equal(got[~nan], want[~nan])
    for x in [dK, dV, cache] + batch + out:
        x.free()
