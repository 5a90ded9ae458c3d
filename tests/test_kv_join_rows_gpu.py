"""Attention over the paged cache with split keys, more than 64 sequences and rows of no sequence before the first one:
every row of every sequence gets its joined sums, the others stay as they were. Against numpy in 64 bits."""
import numpy as np
import pytest

import example_matmul_metal4_amd as mtk  # noqa: F401
from test_kv_cache_use_gpu import Given, agree, rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, dead, chunk, fmt, dtype", [(300, 10, 0, "fp4", "bf16"), (130, 700, 0, "fp8", "f16"), (100, 5, 500, "fp4", "f16")])
def test_rows_before_the_first_sequence(dev, n, dead, chunk, fmt, dtype):
    # more rows than the join has workgroups, so that each has several, the first of them in front of the sequences
    rng = rng_of(80)
    lens = [int(x) for x in rng.integers(300, 1100, n)]
    rows = [1] * n
    rows[7] = 0
    if chunk:
        lens[-1], rows[-1] = 1500, chunk
    g = Given(dev, 81, lens, rows, 32, 8, 128, 16, fmt, dtype, n_pages=200, width=512)
    g.start += dead
    g.T += dead
    g.Q = np.resize(g.Q, (g.T,) + g.Q.shape[1:])
    S_q = 0 if chunk else 1
    d = g.plan(S_q).describe()
    assert "keys split" in d and ("mtk_kv_join_rows" in d or "prefill" in d)
    some = set(range(n + dead)) | {n + dead + 200, int(g.start[-1]) - 1}
    got, lse = g.attend(S_q)
    want, ref, bound = g.cache.attention(g.Q, g.start, g.lens, g.table, True, S_q, some)
    assert (got[:dead] == 0x1234).all() and (lse[:dead] == 77.0).all()
    agree(got, lse, want, ref, bound, dtype, untouched=False)
    g.free()


@pytest.mark.parametrize("D", [72, 96, 136, 160, 192, 224])
@pytest.mark.parametrize("fmt, dtype", [("fp4", "f16"), ("fp8", "bf16")])
def test_joins_over_the_parts_with_lanes_left_over(dev, D, fmt, dtype):
    # head dimensions whose D / 4 lanes do not divide the 256 threads of a join
    g = Given(dev, 85, [9000, 2000, 40], [1, 0, 1], 6, 2, D, 16, fmt, dtype, n_pages=200)
    assert "mtk_kv_join_parts" in g.plan(1).describe()
    g.check(1)
    g.free()
