"""Attention over the paged cache where its weights are far apart: one key far above thousands of others, whose small weights
together still count. Against numpy in 64 bits."""
import numpy as np
import pytest

from oracle import kv
from test_kv_cache_use_gpu import Given, agree, rng_of

pytestmark = pytest.mark.gpu

# (lens, rows, H, H_kv, D, page, fmt, width, kernel): single tokens whole and split, drafts, a chunk whole and split
KERNELS = [
    ([2000, 1100], [1, 1], 8, 2, 128, 16, "fp4", None, "_w16_"),
    ([40000, 900], [1, 1], 4, 1, 128, 64, "fp4", None, "mtk_kv_join_parts"),
    ([9000, 3000], [1, 2], 4, 2, 72, 16, "fp8", 600, "_r1_"),
    ([3000, 1500], [5, 4], 8, 2, 64, 32, "fp4", 1000, "_r2_"),
    ([2500, 1300], [3, 3], 4, 2, 192, 16, "fp8", None, "_d256_"),
    ([1000, 900], [70, 66], 2, 1, 64, 16, "fp4", None, "prefill"),
    ([6000], [90], 4, 2, 128, 64, "fp8", None, "prefill"),
    ([3000], [80], 2, 2, 256, 32, "fp4", None, "prefill"),
]


def set_dim(g, which, keys, dim, value):
    """Dim `dim` of K or V at positions `keys` of every sequence and head to `value`."""
    c, P = g.cache, g.cache.page
    grid, scale = (kv.FP4, 125) if c.fmt == "fp4" else (kv.FP8, 119)  # scales among those that the other blocks have
    code = int(np.flatnonzero(grid * 2.0 ** (scale - 127) == abs(value))[0]) + ((8 if c.fmt == "fp4" else 128) if value < 0 else 0)
    for b, n in enumerate(g.lens):
        pos = np.asarray([k for k in keys if k < n])
        page, off = g.table[b, pos // P], pos % P
        codes, scales = c.part(which, False), c.part(which, True)
        scales[page, :, off, dim // 32] = scale
        if c.fmt == "fp8":
            codes[page, :, off, dim] = code
        else:
            old = codes[page, :, off, dim // 2]
            codes[page, :, off, dim // 2] = (old & 0x0F) | (code << 4) if dim % 2 else (old & 0xF0) | code


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_one_key_far_above_the_others(dev, case, first, dtype):
    # 15 to 18 nats between a sequence's first (or last) position and the others, whose own values lie in a dim of their own
    lens, rows, H, H_kv, D, page, fmt, width, kernel = case
    g = Given(dev, 82, lens, rows, H, H_kv, D, page, fmt, dtype, width=width)
    assert kernel in g.plan(max(rows)).describe()
    T, rng = g.T, rng_of(83)
    most = max(lens)
    top = [0] if first else [n - rows[b] for b, n in enumerate(lens)]
    set_dim(g, 0, range(most), 0, 0.0)
    set_dim(g, 1, range(most), 1, 1.5)
    for b in range(len(lens)):
        one = type("One", (), dict(cache=g.cache, lens=g.lens[b:b + 1], table=g.table[b:b + 1]))
        key = [top[0 if first else b]]
        set_dim(one, 0, key, 0, 1.0)
        set_dim(one, 1, key, 1, 0.0)
    q = rng.standard_normal((T, H, D)) / 16
    q[..., 0] = rng.uniform(15, 18, (T, H)) * np.sqrt(D)
    g.Q = kv.bits_of(q, dtype)
    got, lse = g.attend(max(rows))
    want, ref, bound = g.cache.attention(g.Q, g.start, g.lens, g.table, True, max(rows))
    live = bound[..., 1] >= 0
    assert (np.abs(want[..., 1][live]) > 0).all() and (bound[..., 1][live] < 0.1 * want[..., 1][live]).all()  # the small weights show
    agree(got, lse, want, ref, bound, dtype)
    g.free()
