"""Attention over the paged cache by plans whose schedule has steps of more than 64 keys, as all of their sequences may have many
rows and long tables: chunks whole and split, tokens beside them. Against numpy in 64 bits."""
import numpy as np
import pytest

from test_kv_cache_use_gpu import Given, agree, rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, T, S_q, H, H_kv, D, page, width, chunk, fmt, dtype, split", [
    (256, 4351, 4096, 32, 8, 128, 64, 2048, 300, "fp4", "bf16", False),
    (400, 2000, 2000, 8, 2, 64, 1024, 1 << 12, 250, "fp8", "f16", True),
    (400, 2000, 2000, 8, 2, 256, 256, 1 << 14, 130, "fp4", "f16", True),
])
def test_chunk_beside_tokens(dev, B, T, S_q, H, H_kv, D, page, width, chunk, fmt, dtype, split):
    rng = rng_of(90)
    lens, rows = [int(x) for x in rng.integers(1, 600, B)], [1] * B
    lens[B // 2], rows[B // 2] = 3000, chunk
    lens[5], rows[5] = 90, 70
    rows[6] = 0
    used = sum(-(-n // page) for n in lens)
    g = Given(dev, 91, lens, rows, H, H_kv, D, page, fmt, dtype, n_pages=min(used + 1, 60), width=width)
    g.T = T
    g.Q = np.resize(g.Q, (T,) + g.Q.shape[1:])
    d = g.plan(S_q).describe()
    assert "prefill" in d and ("keys split" in d.split("rows/wg=128")[1]) == split
    at = int(g.start[B // 2])
    some = {0, 4, 5, int(g.start[5]) + 69, at - 1, at, at + chunk // 2, at + chunk - 1, at + chunk, int(g.start[-1]) - 1}
    got, lse = g.attend(S_q)
    want, ref, bound = g.cache.attention(g.Q, g.start, g.lens, g.table, True, S_q, some)
    end = int(g.start[-1])
    assert (got[end:] == 0x1234).all() and (lse[end:] == 77.0).all()
    assert not (lse[:end] == 77.0).any()  # every row was written
    agree(got, lse, want, ref, bound, dtype, untouched=False)
    g.free()
