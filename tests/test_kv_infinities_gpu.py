"""Attention over the paged cache with infinities in Q, where every score of a row is -inf or one is +inf. Against numpy in 64
bits."""
import numpy as np
import pytest

from oracle import kv
from test_kv_cache_use_gpu import Given, agree
from test_kv_weights_gpu import KERNELS, set_dim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_infinite_queries(dev, case, dtype):
    # a row whose scores are all -inf gives NaN, with a log-sum-exp of -inf; one of them +inf: NaN
    lens, rows, H, H_kv, D, page, fmt, width, kernel = case
    g = Given(dev, 84, lens, rows, H, H_kv, D, page, fmt, dtype, width=width)
    set_dim(g, 0, range(max(lens)), 2, 1.0)
    set_dim(g, 0, [0, lens[0] - 2, lens[0] - 1], 3, -0.5)
    x = kv.to_f64(g.Q, dtype).copy()
    for t in range(g.T):
        for h in range(H):
            x[t, h, 2] = (-np.inf, np.inf, x[t, h, 2], x[t, h, 2])[(t + h) % 4]
    x[0, 0, 2], x[0, 0, 3] = 0.5, np.nan
    g.Q = kv.bits_of(x, dtype)
    got, lse = g.attend(max(rows))
    with np.errstate(all="ignore"):
        want, ref, bound = g.cache.attention(g.Q, g.start, g.lens, g.table, True, max(rows))
    row, low = ~(bound[..., 0] < 0), np.isneginf(x[..., 2])
    assert np.isnan(want[row & np.isinf(x[..., 2])]).all() and (row & low).any()
    assert np.isneginf(ref[row & low]).all()
    agree(got, lse, want, ref, np.where(np.isnan(bound), 0.0, bound), dtype)
    g.free()
