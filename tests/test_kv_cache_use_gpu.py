"""The paged key/value cache in few bits as a server uses it: caches with NaN blocks and pages that are none, lengths that
do not fit, large batches and long tables, graphs replayed with other lengths, other streams, and the three operators
together over the steps of a generation. Against numpy in 64 bits (oracle/kv.py)."""
import ctypes

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import kv

pytestmark = pytest.mark.gpu

rng_of = lambda seed: np.random.default_rng(seed)
i32 = lambda x: np.ascontiguousarray(x, np.int32)


class Given:
    """A batch whose pages hold random codes and moderate scales, every byte of them valid; pages may be shared."""

    def __init__(self, dev, seed, lens, rows, H, H_kv, D, page, fmt, dtype, n_pages=None, width=None, table=None):
        rng = rng_of(seed)
        self.dev, self.H, self.dtype = dev, H, dtype
        self.lens, self.start = i32(lens), i32(np.concatenate([[0], np.cumsum(rows)]))
        used = [-(-max(0, n) // page) for n in lens]
        width = width or max(1, max(used))
        n_pages = n_pages or sum(used) + 1
        if table is None:
            order = rng.permutation(n_pages) if sum(used) <= n_pages else None
            table, at = np.full((len(lens), width), -1, np.int32), 0
            for b, n in enumerate(used):
                table[b, :n] = rng.integers(0, n_pages, n) if order is None else order[at:at + n]
                at += n
        self.table = i32(table)
        c = self.cache = kv.Cache(n_pages, page, H_kv, D, fmt, dtype)
        c.bytes[:] = rng.integers(0, 256, c.bytes.size, dtype=np.uint8)
        for w in range(2):
            if fmt == "fp8":  # the two NaN codes are never written
                codes = c.part(w, False)
                codes[(codes & 0x7F) == 0x7F] = 0x3A
            # values of about 1: e2m1 codes are 2 on average, e4m3's are spread over 2^-9 to 448
            scale = c.part(w, True)
            scale[:] = rng.integers(124, 127, scale.shape) if fmt == "fp4" else rng.integers(117, 120, scale.shape)
        self.T = int(self.start[-1]) + 1
        self.Q = kv.bits_of(rng.standard_normal((self.T, H, D)) / 4, dtype)
        self.pages = dict(n_pages=n_pages, page_size=page, max_pages=width, format=fmt, dtype=dtype)
        self.d = None

    def up(self):
        if self.d is None:
            self.d = [self.dev.upload(x) for x in (self.cache.bytes, self.start, self.lens, self.table, self.Q)]
        return self.d

    def plan(self, S_q=0, causal=True):
        return mtk.KvAttentionPlan(self.dev, len(self.lens), self.T, self.H, self.cache.H_kv, self.cache.D, S_q=S_q,
                                   causal=causal, **self.pages)

    def attend(self, S_q=0, causal=True, plan=None):
        dev, (cache, start, lens, table, Q) = self.dev, self.up()
        plan = plan or self.plan(S_q, causal)
        print(plan.describe(), flush=True)
        O, lse = dev.upload(np.full(self.Q.shape, 0x1234, np.uint16)), dev.upload(np.full(self.Q.shape[:2], 77.0, np.float32))
        ws = dev.upload(np.full(plan.workspace_bytes, 0xFF, np.uint8)) if plan.workspace_bytes else None
        plan.run(Q, cache, start, lens, table, O, lse, ws)
        dev.sync()
        got = dev.download(O, self.Q.shape, np.uint16), dev.download(lse, self.Q.shape[:2], np.float32)
        for x in (O, lse, ws):
            if x is not None:
                x.free()
        return got

    def check(self, S_q=0, causal=True, only=None):
        got, lse = self.attend(S_q, causal)
        want, ref, bound = self.cache.attention(self.Q, self.start, self.lens, self.table, causal, S_q, only)
        agree(got, lse, want, ref, bound, self.dtype, untouched=only is None)
        return got, lse

    def free(self):
        for x in self.d or []:
            x.free()


def agree(got, lse, want, ref, bound, dtype, untouched=True):
    free = bound < 0
    if untouched:
        assert (got[free] == 0x1234).all() and (lse[free[..., 0]] == 77.0).all()
    x = kv.to_f64(got, dtype)
    nan = np.isnan(want) & ~free
    assert np.array_equal(np.isnan(x) & ~free, nan)
    use = ~free & ~nan
    off = np.abs(np.where(use, x, 0) - np.where(use, want, 0))
    print(f"worst {(off[use] / np.maximum(bound[use], 1e-300)).max() if use.any() else 0:.3f} of the bound, "
          f"{int(nan.sum())} NaN of {int((~free).sum())}", flush=True)
    assert (off[use] <= bound[use]).all()
    row = ~free[..., 0]
    assert np.array_equal(np.isnan(lse) & row, np.isnan(ref) & row) and np.array_equal(np.isneginf(lse) & row, np.isneginf(ref) & row)
    live = row & np.isfinite(ref)
    # scores as in the bound; the logarithm and its factor: a few steps of 32 bits
    assert (np.abs(lse[live] - ref[live]) <= 2e-5 * (1 + np.abs(ref[live]))).all()


# one of each kernel: 16 wavefronts, 16 / 32 / 64 rows per workgroup, rows over the wavefronts; whole pairs and shared ones
KERNELS = [
    ([170, 93], [1, 1], 8, 2, 128, 16, "fp4", "bf16", "w16"),
    ([170, 93], [1, 1], 8, 2, 64, 32, "fp8", "f16", "w16"),
    ([4500, 93], [1, 2], 8, 2, 128, 16, "fp4", "f16", "_r1_"),
    ([4500, 93], [1, 2], 8, 2, 56, 64, "fp8", "bf16", "_r1_"),
    ([400, 200], [3, 1], 4, 2, 256, 16, "fp4", "f16", "_r1_"),
    ([200, 93], [9, 4], 6, 2, 72, 16, "fp4", "f16", "_r2_"),
    ([1500, 93], [9, 4], 6, 2, 128, 16, "fp8", "bf16", "_r2_"),
    ([1500, 93], [19, 4], 6, 2, 64, 32, "fp4", "bf16", "_r4_"),
    ([300, 93], [19, 4], 6, 2, 128, 16, "fp8", "f16", "_r4_"),
    ([300, 93], [12, 4], 4, 2, 232, 16, "fp4", "bf16", "_r2_"),
    ([300, 93], [120, 4], 4, 2, 64, 16, "fp4", "f16", "prefill"),
    ([900, 93], [120, 4], 4, 2, 64, 16, "fp8", "bf16", "prefill"),
    ([300, 93], [90, 40], 4, 2, 128, 32, "fp4", "bf16", "prefill"),
    ([900, 93], [90, 1], 4, 2, 128, 16, "fp8", "f16", "prefill"),
    ([300, 93], [70, 9], 4, 2, 256, 16, "fp4", "f16", "prefill"),
    ([900, 93], [70, 9], 4, 2, 160, 64, "fp8", "bf16", "prefill"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_nan_blocks(dev, case, causal):
    lens, rows, H, H_kv, D, page, fmt, dtype, kernel = case
    g = Given(dev, 40, lens, rows, H, H_kv, D, page, fmt, dtype)
    assert kernel in g.plan(max(rows), causal).describe()
    c, rng = g.cache, rng_of(41)
    at = lambda b, pos: (int(g.table[b, pos // page]), pos % page)
    for b, n in enumerate(lens):
        # V: any block of any position, the last ones too, which only the last rows see
        for pos in list(rng.integers(0, n, 2)) + [n - 1, max(0, n - rows[b])]:
            p, o = at(b, int(pos))
            c.part(1, True)[p, rng.integers(H_kv), o, rng.integers(c.blocks)] = 255
    # K: the position of the last row of one head of the first sequence; the second's last but one, another head
    p, o = at(0, lens[0] - 1)
    c.part(0, True)[p, 0, o, c.blocks - 1] = 255
    p, o = at(1, lens[1] - 2)
    c.part(0, True)[p, 1, o, 0] = 255
    g.check(max(rows), causal)
    g.free()


@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_pages_that_are_none(dev, case):
    lens, rows, H, H_kv, D, page, fmt, dtype, kernel = case
    for bad in (-1, 1 << 30, -(1 << 31)):
        g = Given(dev, 42, lens + [40, 50, 3, -5, 30], rows + [1, 2, 3, 1, 0], H, H_kv, D, page, fmt, dtype)
        g.lens[4] = 1  # three rows: the first two lie before the sequence's start and see nothing
        g.table[0, (lens[0] - 1) // page] = bad  # seen by the last rows
        g.table[1, 0] = g.cache.n_pages  # seen by every row
        g.lens[3] = g.table.shape[1] * page + 1  # more positions than the table has
        g.check(max(rows))
        out = [dev.upload(np.full((g.T, H_kv, D), 0x1234, np.uint16)) for _ in range(2)]
        r = mtk.KvReadPlan(dev, len(g.lens), g.T, H_kv, D, **g.pages)
        r.run(*g.d[:4], *out)
        w = mtk.KvWritePlan(dev, len(g.lens), g.T, H_kv, D, **g.pages)
        K, V = (kv.bits_of(rng_of(43 + i).standard_normal((g.T, H_kv, D)), dtype) for i in range(2))
        k = [dev.upload(x) for x in (K, V)]
        want = g.cache.read(g.T, g.start, g.lens, g.table, 0x1234)
        dev.sync()
        for x, y in zip(out, want):
            x = dev.download(x, y.shape, np.uint16)
            nan = np.isnan(kv.to_f64(y, dtype))
            assert np.array_equal(np.isnan(kv.to_f64(x, dtype)), nan) and np.array_equal(x[~nan], y[~nan])
        w.run(*k, *g.d[:4])
        g.cache.write(K, V, g.start, g.lens, g.table)
        dev.sync()
        assert np.array_equal(dev.download(g.d[0], g.cache.bytes.shape, np.uint8), g.cache.bytes)
        for x in out + k:
            x.free()
        g.free()


def test_row_starts_out_of_range(dev):
    # limited to [0, T] and to ascend; rows of no sequence are left as they were
    for S_q in (0, 1):
        g = Given(dev, 44, [40, 90, 60, 33], [3, 3, 3, 3], 4, 2, 64, 16, "fp4", "f16")
        g.start[:] = [-7, 2, 2, 6, (1 << 31) - 1]
        g.check(S_q)
        g.free()
    g = Given(dev, 45, [40, 90], [100, 30], 4, 2, 64, 16, "fp4", "f16")
    g.start[:] = [50, 20, 131]  # the first has none; the second one row more than its length allows for, and so on
    g.check()
    g.free()


@pytest.mark.parametrize("rows, S_q, page, width, D, fmt", [
    ("ones", 1, 16, None, 64, "fp4"), ("ones", 1, 32, 400, 64, "fp8"), ("ones", 1, 16, 70, 256, "fp4"),
    ("drafts", 5, 16, 400, 128, "fp4"), ("mixed", 0, 16, None, 64, "fp4"), ("mixed", 0, 64, None, 128, "fp8")])
def test_large_batches(dev, rows, S_q, page, width, D, fmt):
    # more than 64 sequences: the kernels take them 64 at a time; some without rows or positions
    rng = rng_of(46)
    n = 150
    lens = rng.integers(0, 300, n)
    lens[::17] = 0
    count = {"ones": np.ones(n, int), "drafts": rng.integers(0, 6, n), "mixed": np.where(np.arange(n) % 50 == 49, 60, 1)}[rows]
    count = np.minimum(count, lens)
    g = Given(dev, 47, list(lens), list(count), 6, 3, D, page, fmt, "bf16", width=width)
    g.check(S_q)
    g.free()


def test_shared_pages_and_long_tables(dev):
    # tables of more than the 64 entries that a wavefront holds at once, walked by workgroups with long shares; a few
    # pages for all of them
    rng = rng_of(48)
    lens = [int(x) for x in rng.integers(3500, 4300, 40)]
    g = Given(dev, 49, lens, [1] * 40, 8, 8, 64, 16, "fp4", "f16", n_pages=60, width=300)
    g.check(1)
    g.free()
    lens = [3900] + [100] * 14 + [2000]
    g = Given(dev, 50, lens, [1] * 16, 8, 8, 128, 16, "fp8", "bf16", n_pages=30)
    assert "_w16_" in g.plan(1).describe()
    g.check(1)
    g.free()
    # rows over the wavefronts, the keys of every pair in one workgroup
    g = Given(dev, 51, [3000, 1500], [1500, 900], 32, 8, 64, 16, "fp4", "f16", n_pages=40)
    d = g.plan().describe()
    assert "prefill" in d and "keys split" not in d.split("rows/wg=128")[1]
    g.check(only={0, 1, 700, 1499, 1500, 2399})
    g.free()


@pytest.mark.parametrize("tokens, D, fmt, dtype", [(3, 64, "fp4", "f16"), (70, 64, "fp8", "bf16"), (9, 256, "fp4", "bf16")])
def test_tokens_beside_a_chunk(dev, tokens, D, fmt, dtype):
    # single tokens whose keys are split, joined in the chunk's launch; a chunk whose keys are split; one in the middle of the
    # batch, rows of no sequence between
    rng = rng_of(54)
    half = tokens // 2
    lens = [int(x) for x in rng.integers(900, 1400, half)] + [1500] + [int(x) for x in rng.integers(1, 1400, tokens - half)]
    g = Given(dev, 55, lens, [1] * half + [80] + [1] * (tokens - half), 8, 2, D, 16, fmt, dtype, n_pages=100, width=300)
    d = g.plan().describe()
    assert "prefill" in d and d.count("keys split") == 2 and d.count("join") == 1
    g.check()
    g.free()


def test_offsets_past_32_bits(dev):
    # pages whose bytes lie past 2^32 in the cache: 280000 of 17408 bytes, 4.9 GB
    H_kv, D, page = 8, 128, 16
    size = mtk.kv_cache_bytes(1, page, H_kv, D)
    n_pages = 280000
    g = Given(dev, 52, [40, 33], [2, 1], 16, H_kv, D, page, "fp4", "bf16", n_pages=6)
    far = i32(np.where(g.table >= 0, g.table + n_pages - 6, -1))
    cache = dev.empty(n_pages * size)
    print("cache of", cache.nbytes, "bytes", flush=True)
    assert (n_pages - 6) * size > 1 << 32
    at = cache.ptr + (n_pages - 6) * size
    tail = mtk.DeviceBuffer(dev, at, 6 * size)
    dev.upload_into(tail, g.cache.bytes)
    pages = {**g.pages, "n_pages": n_pages}
    d = [dev.upload(x) for x in (g.start, g.lens, far, g.Q)]
    K, V = (kv.bits_of(rng_of(53 + i).standard_normal((g.T, H_kv, D)), "bf16") for i in range(2))
    k = [dev.upload(x) for x in (K, V)]
    O, lse = dev.upload(np.full(g.Q.shape, 0x1234, np.uint16)), dev.upload(np.full(g.Q.shape[:2], 77.0, np.float32))
    back = [dev.upload(np.full(K.shape, 0x1234, np.uint16)) for _ in range(2)]
    mtk.KvWritePlan(dev, 2, g.T, H_kv, D, **pages).run(*k, cache, *d[:3])
    mtk.KvAttentionPlan(dev, 2, g.T, 16, H_kv, D, S_q=2, **pages).run(d[3], cache, *d[:3], O, lse)
    mtk.KvReadPlan(dev, 2, g.T, H_kv, D, **pages).run(cache, *d[:3], *back)
    dev.sync()
    g.cache.write(K, V, g.start, g.lens, g.table)
    assert np.array_equal(dev.download(tail, g.cache.bytes.shape, np.uint8), g.cache.bytes)
    want, ref, bound = g.cache.attention(g.Q, g.start, g.lens, g.table)
    agree(dev.download(O, g.Q.shape, np.uint16), dev.download(lse, g.Q.shape[:2], np.float32), want, ref, bound, "bf16")
    for x, y in zip(back, g.cache.read(g.T, g.start, g.lens, g.table, 0x1234)):
        assert np.array_equal(dev.download(x, y.shape, np.uint16), y)
    for x in [cache, O, lse] + d + k + back:
        x.free()


# ------------------------------------------------------------------ graphs, streams, several runs at once

def test_graphs_replayed_with_other_lengths(dev):
    # one graph of each operator serves every step: the lengths, the table and the rows lie on the device
    H, H_kv, D, page, B = 6, 2, 96, 16, 3
    width, n_pages = 300, 40
    c = kv.Cache(n_pages, page, H_kv, D, "fp4", "bf16")
    pages = dict(n_pages=n_pages, page_size=page, max_pages=width, format="fp4", dtype="bf16")
    rng, T = rng_of(60), 8
    cache = dev.upload(c.bytes)
    start, lens, table = (dev.empty(4 * n) for n in (B + 1, B, B * width))
    K, V, Q, O = (dev.empty(2 * T * h * D) for h in (H_kv, H_kv, H, H))
    back = [dev.empty(2 * T * H_kv * D) for _ in range(2)]
    lse = dev.empty(4 * T * H)
    w = mtk.KvWritePlan(dev, B, T, H_kv, D, **pages)
    r = mtk.KvReadPlan(dev, B, T, H_kv, D, **pages)
    a = mtk.KvAttentionPlan(dev, B, T, H, H_kv, D, S_q=4, **pages)
    assert "keys split" in a.describe()
    ws = dev.empty(a.workspace_bytes)
    graphs = [w.graph([w.args(K, V, cache, start, lens, table)], 1), a.graph([a.args(Q, cache, start, lens, table, O, lse, ws)], 1),
              r.graph([r.args(cache, start, lens, table, *back)], 1)]
    order = rng.permutation(n_pages)
    t = np.full((B, width), -1, np.int32)
    t[0, :20], t[1, :3], t[2, :10] = order[:20], order[20:23], order[23:33]
    now = np.zeros(B, int)
    try:
        for step, rows in enumerate([(4, 0, 1), (1, 4, 1), (0, 0, 0), (2, 2, 3), (4, 4, 0)]):
            grow = (0, 30, 100, 0, 60)[step]  # a jump in the first sequence's length: positions that nothing was written to
            now = now + np.array(rows) + np.array([grow, 0, 0])
            s = i32(np.concatenate([[0], np.cumsum(rows)]))
            k, v = (kv.bits_of(rng.standard_normal((T, H_kv, D)), "bf16") for _ in range(2))
            q = kv.bits_of(rng.standard_normal((T, H, D)), "bf16")
            for buf, x in ((start, s), (lens, i32(now)), (table, t), (K, k), (V, v), (Q, q)):
                dev.upload_into(buf, x)
            for buf, n in ((O, T * H * D), (back[0], T * H_kv * D), (back[1], T * H_kv * D)):
                dev.upload_into(buf, np.full(n, 0x1234, np.uint16))
            dev.upload_into(lse, np.full(T * H, 77.0, np.float32))
            for g in graphs:
                g.launch()
            dev.sync()
            c.write(k, v, s, now, t)
            assert np.array_equal(dev.download(cache, c.bytes.shape, np.uint8), c.bytes), step
            want, ref, bound = c.attention(q, s, now, t, S_q=4)
            agree(dev.download(O, q.shape, np.uint16), dev.download(lse, (T, H), np.float32), want, ref, bound, "bf16")
            for x, y in zip(back, c.read(T, s, now, t, 0x1234)):
                assert np.array_equal(dev.download(x, y.shape, np.uint16), y), step
    finally:
        for g in graphs:
            g.close()
    for x in [cache, start, lens, table, K, V, Q, O, lse, ws] + back:
        x.free()


def test_other_streams_and_captures(dev):
    g = Given(dev, 62, [5000, 300], [1, 90], 8, 2, 128, 16, "fp4", "f16")
    plan = g.plan()
    ref, ref_lse = g.check()
    cache, start, lens, table, Q = g.up()
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    streams = [ctypes.c_void_p() for _ in range(2)]
    outs = [(dev.empty(ref.nbytes), dev.empty(ref_lse.nbytes), dev.empty(plan.workspace_bytes)) for _ in range(2)]
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    live = np.arange(g.T) < g.start[-1]

    def poison():
        for o, l, ws in outs:
            dev.upload_into(o, np.full(ref.shape, 0x7E00, np.uint16))
            dev.upload_into(l, np.zeros(ref_lse.shape, np.float32))
            dev.upload_into(ws, np.full(ws.nbytes, 0xFF, np.uint8))

    def same(which):
        assert hip.hipDeviceSynchronize() == 0
        for o, l, _ in which:
            assert np.array_equal(dev.download(o, ref.shape, np.uint16)[live], ref[live])
            assert np.array_equal(dev.download(l, ref_lse.shape, np.float32)[live], ref_lse[live])

    try:
        for s in streams:
            assert hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0  # non-blocking
        for _ in range(3):  # two runs at once, each with its own workspace
            poison()
            dev.sync()
            for s, (o, l, ws) in zip(streams, outs):
                mtk._check(mtk.lib().mtk_set_stream(dev.handle, s))
                plan.run(Q, cache, start, lens, table, o, l, ws)
            same(outs)
        # two runs in one caller's capture that share a workspace: one after the other on one stream
        mtk._check(mtk.lib().mtk_set_stream(dev.handle, streams[0]))
        assert hip.hipStreamBeginCapture(streams[0], 2) == 0  # relaxed
        for o, l, _ in outs:
            plan.run(Q, cache, start, lens, table, o, l, outs[0][2])
        assert hip.hipStreamEndCapture(streams[0], ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(3):
            poison()
            dev.sync()
            assert hip.hipGraphLaunch(graph_exec, streams[0]) == 0
            same(outs)
    finally:
        mtk._check(mtk.lib().mtk_set_stream(dev.handle, None))
        for destroy, x in [("hipGraphExecDestroy", graph_exec), ("hipGraphDestroy", graph)] + [("hipStreamDestroy", s) for s in streams]:
            if x:
                getattr(hip, destroy)(x)
    for x in [x for o in outs for x in o]:
        x.free()
    g.free()


def test_profile(dev):
    g = Given(dev, 64, [900, 300], [1, 90], 8, 2, 128, 16, "fp4", "f16")
    cache, start, lens, table, Q = g.up()
    plan = g.plan()
    O, ws = dev.empty(g.Q.nbytes), dev.empty(max(1, plan.workspace_bytes))
    t = plan.profile([plan.args(Q, cache, start, lens, table, O, None, ws)], warmup=1, iters=3)
    print(t, flush=True)
    assert t["total_ms"] > 0 and len(t["kernels"]) == len(plan.describe().split("kernels: ")[1].split())
    flops, nbytes = plan.work()
    assert flops > 0 and nbytes > 0
    for x in (O, ws):
        x.free()
    g.free()


# ------------------------------------------------------------------ a generation

@pytest.mark.parametrize("fmt, dtype, H, H_kv, D, page", [("fp4", "bf16", 8, 2, 128, 16), ("fp8", "f16", 4, 4, 80, 32)])
def test_generation(dev, fmt, dtype, H, H_kv, D, page):
    # prompts in chunks beside sequences that take single tokens, then drafts; every step writes its rows and attends; at the
    # end each prefix is read back, and attention over it in 16 bits (the framework's, [B][S][H][D]) agrees
    rng, B, width = rng_of(70), 3, 12
    n_pages = 20
    c = kv.Cache(n_pages, page, H_kv, D, fmt, dtype)
    c.bytes[:] = 0xFF  # never written: NaN, if it were used
    pages = dict(n_pages=n_pages, page_size=page, max_pages=width, format=fmt, dtype=dtype)
    cache, table = dev.upload(c.bytes), np.full((B, width), -1, np.int32)
    free = list(rng.permutation(n_pages))
    now = np.zeros(B, int)
    ld = (H + 2 * H_kv) * D
    last = None
    for rows in [(90, 1, 0), (7, 1, 1), (1, 1, 1), (5, 5, 60), (1, 1, 1), (3, 2, 1)]:
        T = sum(rows)
        now = now + rows
        for b in range(B):
            for p in range(-(-int(now[b]) // page)):
                if table[b, p] < 0:
                    table[b, p] = free.pop()
        start = i32(np.concatenate([[0], np.cumsum(rows)]))
        qkv = kv.bits_of(rng.standard_normal((T, H + 2 * H_kv, D)), dtype)
        d = dev.upload(qkv)
        b3 = [dev.upload(x) for x in (start, i32(now), table)]
        at = lambda heads: d.ptr + 2 * heads * D
        mtk.KvWritePlan(dev, B, T, H_kv, D, ld_k=ld, ld_v=ld, **pages).run(at(H), at(H + H_kv), cache, *b3)
        plan = mtk.KvAttentionPlan(dev, B, T, H, H_kv, D, ld_q=ld, **pages)
        print(rows, plan.describe(), flush=True)
        O, lse = dev.empty(2 * T * H * D), dev.empty(4 * T * H)
        ws = dev.empty(max(1, plan.workspace_bytes))
        plan.run(d, cache, *b3, O, lse, ws if plan.workspace_bytes else None)
        dev.sync()
        q = np.ascontiguousarray(qkv[:, :H])
        c.write(qkv[:, H:H + H_kv], qkv[:, H + H_kv:], start, now, table)
        want, ref, bound = c.attention(q, start, now, table)
        got = dev.download(O, q.shape, np.uint16)
        agree(got, dev.download(lse, (T, H), np.float32), want, ref, bound, dtype)
        last = q, got, start, bound
        for x in b3 + [d, O, lse, ws]:
            x.free()
    assert np.array_equal(dev.download(cache, c.bytes.shape, np.uint8), c.bytes)
    total = int(now.sum())
    whole = [dev.upload(x) for x in (i32(np.concatenate([[0], np.cumsum(now)])), i32(now), table)]
    K, V = dev.empty(2 * total * H_kv * D), dev.empty(2 * total * H_kv * D)
    mtk.KvReadPlan(dev, B, total, H_kv, D, **pages).run(cache, *whole, K, V)
    dev.sync()
    K, V = (dev.download(x, (total, H_kv, D), np.uint16) for x in (K, V))
    q, got, start, bound = last
    as_ = (lambda x: x.view(np.float16)) if dtype == "f16" else (lambda x: x)
    for b in range(B):
        s = slice(int(now[:b].sum()), int(now[:b + 1].sum()))
        n = int(start[b + 1] - start[b])
        if n != 1:
            continue  # the 16-bit operator's causal mask starts at the first key
        o = mtk.attention(dev, as_(q[start[b]:start[b] + 1][None]), as_(K[s][None]), as_(V[s][None]), dtype=dtype)
        o = np.ascontiguousarray(o).view(np.uint16)[0]
        i = int(start[b])
        # both are within the bound of the exact result
        assert (np.abs(kv.to_f64(o, dtype) - kv.to_f64(got[i:i + 1], dtype)) <= 2 * bound[i:i + 1]).all()
    for x in whole + [cache]:
        x.free()
