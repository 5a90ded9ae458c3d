"""Products grouped by expert and in 4 bits as a program uses them: every kernel that a plan chooses, a layer of experts forward and
backward, layers held in 4 bits, graphs replayed with other routings, other streams, operands past 2^32 bytes. Against numpy in
64 bits (oracle/experts.py)."""
import ctypes
import functools

import numpy as np
import pytest

import example_matmul_metal4_amd as mtk
from oracle import experts, kv

pytestmark = pytest.mark.gpu

rng_of = lambda seed: np.random.default_rng(seed)
i32 = lambda x: np.ascontiguousarray(x, np.int32)
FILL = 0x1234


def bits(rng, shape, dtype, size=1.0):
    return kv.bits_of(rng.standard_normal(shape) * size, dtype)


def agree(got, want, bound, what):
    off = np.abs(got - want)
    print(f"{what}: worst {(off / np.maximum(bound, 1e-300)).max() if off.size else 0:.3f} of the bound", flush=True)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])


def free(*buffers):
    for b in buffers:
        if b is not None:
            b.free()


def routing(rng, T, E):
    """row_start [E + 1] of ascending groups, some without a row, and rows of none before and behind them."""
    cuts = np.sort(rng.integers(0, T + 1, E + 1))
    if rng.integers(2):
        cuts[0], cuts[E] = 0, T
    return i32(cuts)


# ------------------------------------------------------------------ every kernel

DTYPES = ("f16", "bf16")
KINDS = ["256", "128"] + [f"64{a}_w{w}" for a in ("", "_any") for w in (8, 4, 1)]
FORWARD = [f"mtk_grouped_{dt}_{lay}_{k}" for dt in DTYPES for lay in ("nt", "nn") for k in KINDS]
GRADIENT = [f"mtk_grouped_{dt}_grad_{k}" for dt in DTYPES for k in KINDS]
FEW_BITS = [f"mtk_mx_gemm_{dt}_{k}" for dt in DTYPES for k in ("256", "128", "64", "32", "32q")]


@functools.lru_cache(None)
def shapes():
    """For each kernel the smallest of some thousand problems whose plans choose it, and the smallest with rows of 100 and more."""
    rng, found = rng_of(1), {}

    def size(most):
        return int(np.exp(rng.uniform(0, np.log(most))))

    def take(plan, problem, work):
        name = plan.describe().split("kernels: ")[1].split()
        for n in name:
            if n.startswith("mtk_grouped") or n.startswith("mtk_mx_gemm"):
                at = found.setdefault(n, {})
                for wide in (False, N >= 100 and K >= 100):
                    at[wide] = min(at.get(wide, (work, problem)), (work, problem))

    for i in range(8000):
        E, T, N, K = size(130), size(9000), size(9000), size(5000)
        dt, trans, odd = DTYPES[i & 1], bool(i & 2), i % 3 == 0
        if not odd:
            N, K = N + N % 2, K + K % 2
        work = T * N * K + E * N * K
        if work > 1e11 or (T + E * K) * N > 5e7 or (E * N + T) * K > 5e7:
            continue
        take(mtk.GroupedGemmPlan(None, E, T, N, K, trans_b=trans, dtype=dt), (E, T, N, K, trans, dt), work)
        take(mtk.GroupedGradPlan(None, E, T, N, K, trans_b=trans, dtype=dt, out_f32=i % 5 < 2), (E, T, N, K, trans, dt, i % 5 < 2), work)
        groups = E if i & 4 else 0
        take(mtk.MxGemmPlan(None, T, N, K, E=groups, dtype=dt, quantize_a=bool(i & 8)), (groups, T, N, K, dt, bool(i & 8)), work)
    return {n: sorted(set(x.values())) for n, x in found.items()}


@pytest.mark.parametrize("kernel", FORWARD)
def test_forward_kernels(dev, kernel):
    for n, (_, (E, T, N, K, trans_b, dtype)) in enumerate(shapes()[kernel]):
        rng = rng_of(20 + n)
        A, B = bits(rng, (T, K), dtype), bits(rng, (E, N, K) if trans_b else (E, K, N), dtype, K ** -0.5)
        bias, starts = bits(rng, (E, N), dtype), routing(rng, T, E)
        plan = mtk.GroupedGemmPlan(dev, E, T, N, K, trans_b=trans_b, dtype=dtype, has_bias=True)
        print(plan.describe(), flush=True)
        assert kernel in plan.describe()
        d = [dev.upload(x) for x in (A, B, bias, starts, np.full((T + 1, N), FILL, np.uint16))]
        plan.run(*d)
        dev.sync()
        got = dev.download(d[4], (T + 1, N), np.uint16)
        want, bound, mine = experts.grouped(A, B, bias, starts, trans_b, dtype)
        assert (got[:T][~mine] == FILL).all() and (got[T] == FILL).all()
        agree(kv.to_f64(got[:T], dtype)[mine], want[mine], bound[mine], "C")
        free(*d)


@pytest.mark.parametrize("kernel", GRADIENT)
def test_gradient_kernels(dev, kernel):
    for n, (_, (E, T, N, K, trans_b, dtype, out_f32)) in enumerate(shapes()[kernel]):
        rng = rng_of(30 + n)
        A, dC, starts = bits(rng, (T, K), dtype), bits(rng, (T, N), dtype), routing(rng, T, E)
        plan = mtk.GroupedGradPlan(dev, E, T, N, K, trans_b=trans_b, dtype=dtype, has_bias=True, out_f32=out_f32)
        print(plan.describe(), flush=True)
        assert kernel in plan.describe()
        kind = np.float32 if out_f32 else np.uint16
        shape = (E, N, K) if trans_b else (E, K, N)
        d = [dev.upload(x) for x in (A, dC, starts, np.full(E * N * K + 64, 7, kind), np.full(E * N + 64, 7, kind))]
        plan.run(*d)
        dev.sync()
        dB, db = dev.download(d[3], (E * N * K + 64,), kind), dev.download(d[4], (E * N + 64,), kind)
        assert (dB[E * N * K:] == 7).all() and (db[E * N:] == 7).all()
        (w, wb), (b, bb) = experts.grad(A, dC, starts, trans_b, dtype, "f32" if out_f32 else dtype)
        val = (lambda x: x.astype(np.float64)) if out_f32 else (lambda x: kv.to_f64(x, dtype))
        agree(val(dB[:E * N * K].reshape(shape)), w, wb, "dB")
        agree(val(db[:E * N].reshape(E, N)), b, bb, "dbias")
        free(*d)


@pytest.mark.parametrize("kernel", FEW_BITS)
def test_few_bit_kernels(dev, kernel):
    for n, (_, (E, T, N, K, dtype, quantize_a)) in enumerate(shapes()[kernel]):
        rng, groups = rng_of(40 + n), max(1, E)
        A, W, bias = bits(rng, (T, K), dtype), bits(rng, (groups * N, K), dtype, K ** -0.5), bits(rng, (groups, N), dtype)
        qa, qb, starts = experts.quantise(A, dtype), experts.quantise(W, dtype), routing(rng, T, E) if E else None
        plan = mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, has_bias=True, quantize_a=quantize_a)
        print(plan.describe(), flush=True)
        assert kernel in plan.describe().split()
        d = [dev.upload(A if quantize_a else qa[0]), None if quantize_a else dev.upload(qa[1]), dev.upload(qb[0]), dev.upload(qb[1]), dev.upload(bias),
             dev.upload(starts) if E else None, dev.upload(np.full((T + 1, N), FILL, np.uint16)), dev.empty(max(16, plan.workspace_bytes))]
        plan.run(*d)
        dev.sync()
        got = dev.download(d[6], (T + 1, N), np.uint16)
        want, bound, mine = experts.mx_product(experts.values(*qa, K), experts.values(*qb, K).reshape(groups, N, K), bias,
                                               starts if E else [0, T], dtype)
        assert (got[:T][~mine] == FILL).all() and (got[T] == FILL).all()
        agree(kv.to_f64(got[:T], dtype)[mine], want[mine], bound[mine], "C")
        free(*d)


@functools.lru_cache(None)
def halved():
    """For each operator's 256 x 256 kernel the smallest of some problems of which the last round's tiles are half of the grid or fewer, so
    that two workgroups share each."""
    rng, found = rng_of(2), {}
    size = lambda least, most: int(np.exp(rng.uniform(np.log(least), np.log(most))))
    up = lambda x: -(-x // 256)
    for i in range(20000):
        E, T, N, K = size(1, 8), size(300, 9000), size(500, 9000), size(65, 6000) & ~1
        N -= N % 2 if i % 3 else 0
        if T * N * K > 1e11 or T * N > 3e7 or E * N * K > 6e7:
            continue
        starts = np.sort(np.r_[0, rng.integers(0, T + 1, E - 1), T])
        blocks = sum(up(b - a) for a, b in zip(starts[:-1], starts[1:]))
        dtype = DTYPES[i & 1]
        makers = {"nt": (lambda: mtk.GroupedGemmPlan(None, E, T, N, K, dtype=dtype), blocks * up(N)),
                  "nn": (lambda: mtk.GroupedGemmPlan(None, E, T, N, K, trans_b=False, dtype=dtype), blocks * up(N)),
                  "grad": (lambda: mtk.GroupedGradPlan(None, E, T, N, K, dtype=dtype, out_f32=bool(i & 4)), E * up(N) * up(K)),
                  "mx": (lambda: mtk.MxGemmPlan(None, T, N, K, E=E, dtype=dtype), blocks * up(N))}
        for kind, (make, total) in makers.items():
            if 0 < total % 256 <= 128 and make().describe().split("kernels: ")[1].endswith("_256"):
                found[kind] = min(found.get(kind, (1e30,)), (T * N * K, i, E, T, N, K, dtype, tuple(starts.tolist()), bool(i & 4)))
    return found


@pytest.mark.parametrize("kind", ["nt", "nn", "grad", "mx"])
def test_tiles_halved(dev, kind):
    _, i, E, T, N, K, dtype, starts, out_f32 = halved()[kind]
    rng, starts = rng_of(90), i32(starts)
    A, bias = bits(rng, (T, K), dtype), bits(rng, (E, N), dtype)
    if kind == "grad":
        dC = bits(rng, (T, N), dtype)
        plan = mtk.GroupedGradPlan(dev, E, T, N, K, dtype=dtype, out_f32=out_f32)
        d = [dev.upload(x) for x in (A, dC, starts)] + [dev.empty((4 if out_f32 else 2) * E * N * K)]
        want, bound = experts.grad(A, dC, starts, True, dtype, "f32" if out_f32 else dtype)[0]
        args, shape = d, (E, N, K)
    elif kind == "mx":
        qa, qb = experts.quantise(A, dtype), experts.quantise(bits(rng, (E * N, K), dtype), dtype)
        plan = mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, has_bias=True)
        d = [dev.upload(x) for x in (*qa, *qb, bias, starts)] + [dev.empty(2 * T * N)]
        want, bound, _ = experts.mx_product(experts.values(*qa, K), experts.values(*qb, K).reshape(E, N, K), bias, starts, dtype)
        args, shape = d, (T, N)
    else:
        B = bits(rng, (E, N, K) if kind == "nt" else (E, K, N), dtype)
        plan = mtk.GroupedGemmPlan(dev, E, T, N, K, trans_b=kind == "nt", dtype=dtype, has_bias=True)
        d = [dev.upload(x) for x in (A, B, bias, starts)] + [dev.empty(2 * T * N)]
        want, bound, _ = experts.grouped(A, B, bias, starts, kind == "nt", dtype)
        args, shape = d, (T, N)
    print(plan.describe(), flush=True)
    assert "_256" in plan.describe()
    plan.run(*args)
    dev.sync()
    f32 = kind == "grad" and out_f32
    got = dev.download(d[-1], shape, np.float32 if f32 else np.uint16)
    agree(got.astype(np.float64) if f32 else kv.to_f64(got, dtype), want, bound, kind)
    free(*d)


# ------------------------------------------------------------------ layers

class Layer:
    """Experts of two products with a bias each over rows sorted by expert, X -> H -> Y, and its gradients, on device buffers."""

    def __init__(self, dev, E, T, D, F, dtype, seed):
        rng = rng_of(seed)
        self.dev, self.E, self.T, self.D, self.F, self.dtype = dev, E, T, D, F, dtype
        self.w1, self.b1 = bits(rng, (E, F, D), dtype, D ** -0.5), bits(rng, (E, F), dtype)
        self.w2, self.b2 = bits(rng, (E, D, F), dtype, F ** -0.5), bits(rng, (E, D), dtype)
        up = dev.upload
        self.d = {n: up(getattr(self, n)) for n in ("w1", "b1", "w2", "b2")}
        for n, width in (("X", D), ("H", F), ("Y", D), ("dY", D), ("dH", F), ("dX", D)):
            self.d[n] = dev.empty(2 * T * width)
        for n, size in (("dw1", E * F * D), ("db1", E * F), ("dw2", E * D * F), ("db2", E * D)):
            self.d[n] = dev.empty(4 * size)
        self.d["starts"] = dev.empty(4 * (E + 1))
        mk = lambda N, K, **kw: mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype, **kw)
        gr = lambda N, K: mtk.GroupedGradPlan(dev, E, T, N, K, dtype=dtype, has_bias=True, out_f32=True)
        d, s = self.d, self.d["starts"]
        self.steps = [(p, p.args(*a)) for p, a in (
            (mk(F, D, has_bias=True), (d["X"], d["w1"], d["b1"], s, d["H"])),
            (mk(D, F, has_bias=True), (d["H"], d["w2"], d["b2"], s, d["Y"])),
            (mk(F, D, trans_b=False), (d["dY"], d["w2"], None, s, d["dH"])),
            (gr(D, F), (d["H"], d["dY"], s, d["dw2"], d["db2"])),
            (mk(D, F, trans_b=False), (d["dH"], d["w1"], None, s, d["dX"])),
            (gr(F, D), (d["X"], d["dH"], s, d["dw1"], d["db1"])))]

    def give(self, X, dY, starts):
        self.X, self.dY, self.starts = X, dY, i32(starts)
        for n in ("X", "dY", "starts"):
            self.dev.upload_into(self.d[n], getattr(self, n))
        for n, width in (("H", self.F), ("Y", self.D), ("dH", self.F), ("dX", self.D)):
            self.dev.upload_into(self.d[n], np.full((self.T, width), FILL, np.uint16))
        for n, b in self.d.items():
            if n in ("dw1", "db1", "dw2", "db2"):
                self.dev.upload_into(b, np.full(b.nbytes // 4, np.nan, np.float32))

    def run(self):
        for p, a in self.steps:
            p.launch(a)

    def got(self, n):
        shape = {"dw1": (self.E, self.F, self.D), "dw2": (self.E, self.D, self.F), "db1": (self.E, self.F), "db2": (self.E, self.D)}.get(n)
        if shape:
            return self.dev.download(self.d[n], shape, np.float32)
        return self.dev.download(self.d[n], (self.T, self.F if n in ("H", "dH") else self.D), np.uint16)

    def check(self):
        """Each operator's output, given those of the operators before it."""
        self.dev.sync()
        H, Y, dH, dX = (self.got(n) for n in ("H", "Y", "dH", "dX"))
        for what, out, (want, bound, mine) in (
                ("H", H, experts.grouped(self.X, self.w1, self.b1, self.starts, True, self.dtype)),
                ("Y", Y, experts.grouped(H, self.w2, self.b2, self.starts, True, self.dtype)),
                ("dH", dH, experts.grouped(self.dY, self.w2, None, self.starts, False, self.dtype)),
                ("dX", dX, experts.grouped(dH, self.w1, None, self.starts, False, self.dtype))):
            assert (out[~mine] == FILL).all(), what
            agree(kv.to_f64(out, self.dtype)[mine], want[mine], bound[mine], what)
        for w, b, x, g in (("dw2", "db2", H, self.dY), ("dw1", "db1", self.X, dH)):
            dw, db = experts.grad(x, g, self.starts, True, self.dtype, "f32")
            agree(self.got(w).astype(np.float64), *dw, w)
            agree(self.got(b).astype(np.float64), *db, b)

    def close(self):
        free(*self.d.values())


@pytest.mark.parametrize("E, T, D, F, dtype", [(8, 96, 256, 384, "bf16"), (5, 33, 75, 130, "f16"), (12, 1500, 512, 1100, "f16"), (3, 1, 64, 128, "bf16")])
def test_expert_layer(dev, E, T, D, F, dtype):
    layer, rng = Layer(dev, E, T, D, F, dtype, 50), rng_of(51)
    for starts in (np.linspace(0, T, E + 1).round(), routing(rng, T, E)):
        layer.give(bits(rng, (T, D), dtype), bits(rng, (T, D), dtype), starts)
        layer.run()
        layer.check()
    layer.close()


def test_graphs_replayed_with_other_routings(dev):
    # one graph of each operator serves every routing: row_start and the rows lie on the device
    for E, T, D, F, dtype in ((6, 120, 96, 200, "bf16"), (70, 300, 77, 90, "f16"), (4, 2500, 640, 2560, "bf16")):
        layer, rng = Layer(dev, E, T, D, F, dtype, 52), rng_of(53)
        graphs = [p.graph([a], 1) for p, a in layer.steps]
        try:
            for starts in (np.zeros(E + 1), routing(rng, T, E), np.linspace(0, T, E + 1).round(), [0] + [T] * E, [T // 3] * E + [T]):
                layer.give(bits(rng, (T, D), dtype), bits(rng, (T, D), dtype), starts)
                for g in graphs:
                    g.launch()
                dev.sync()
                replayed = {n: layer.got(n) for n in ("H", "Y", "dH", "dX", "dw1", "db1", "dw2", "db2")}
                layer.check()
                layer.give(layer.X, layer.dY, layer.starts)  # and eager work between the replays, the same bits
                layer.run()
                dev.sync()
                assert all(np.array_equal(layer.got(n), x) for n, x in replayed.items())
        finally:
            for g in graphs:
                g.close()
        layer.close()


class Held:
    """A layer whose weights lie in 4 bits, brought there by the operator, and whose rows the run brings there."""

    def __init__(self, dev, E, T, N, K, dtype, seed):
        rng, groups = rng_of(seed), max(1, E)
        self.dev, self.E, self.T, self.N, self.K, self.dtype = dev, E, T, N, K, dtype
        W = bits(rng, (groups * N, K), dtype, K ** -0.5)
        self.bias = bits(rng, (groups, N), dtype)
        want = experts.quantise(W, dtype)
        w, self.codes, self.scales = dev.upload(W), dev.empty(want[0].nbytes), dev.empty(want[1].nbytes)
        mtk.MxQuantizePlan(dev, groups * N, K, dtype=dtype).run(w, self.codes, self.scales)
        dev.sync()
        assert np.array_equal(dev.download(self.codes, want[0].shape, np.uint8), want[0])
        assert np.array_equal(dev.download(self.scales, want[1].shape, np.uint8), want[1])
        self.weights = experts.values(*want, K).reshape(groups, N, K)
        self.d_bias = dev.upload(self.bias)
        self.plan = mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, has_bias=True, quantize_a=True)
        print(self.plan.describe(), flush=True)
        free(w)

    def args(self, A, starts, C, workspace):
        return self.plan.args(A, None, self.codes, self.scales, self.d_bias, starts if self.E else None, C, workspace)

    def check(self, A, starts, got):
        v = experts.values(*experts.quantise(A, self.dtype), self.K)
        want, bound, mine = experts.mx_product(v, self.weights, self.bias, starts if self.E else [0, self.T], self.dtype)
        assert (got[~mine] == FILL).all()
        agree(kv.to_f64(got, self.dtype)[mine], want[mine], bound[mine], "C")

    def close(self):
        free(self.codes, self.scales, self.d_bias)


@pytest.mark.parametrize("E, T, D, F, dtype", [(0, 1, 256, 700, "bf16"), (0, 40, 300, 512, "f16"), (8, 60, 256, 320, "bf16"),
                                               (0, 2000, 520, 1030, "f16"), (5, 900, 400, 2050, "bf16")])
def test_layers_in_4_bits(dev, E, T, D, F, dtype):
    # two layers one after the other, as graphs replayed with other rows and routings, each with a workspace of its own
    rng, groups = rng_of(60), max(1, E)
    up, down = Held(dev, E, T, F, D, dtype, 61), Held(dev, E, T, D, F, dtype, 62)
    X, H, Y, s = dev.empty(2 * T * D), dev.empty(2 * T * F), dev.empty(2 * T * D), dev.empty(4 * (groups + 1))
    ws = [dev.empty(max(16, h.plan.workspace_bytes)) for h in (up, down)]
    graphs = [up.plan.graph([up.args(X, s, H, ws[0])], 1), down.plan.graph([down.args(H, s, Y, ws[1])], 1)]
    try:
        for step in range(3):
            x, starts = bits(rng, (T, D), dtype), routing(rng, T, groups)
            dev.upload_into(X, x)
            dev.upload_into(s, starts)
            dev.upload_into(H, np.full((T, F), FILL, np.uint16))
            dev.upload_into(Y, np.full((T, D), FILL, np.uint16))
            for g in graphs:
                g.launch()
            dev.sync()
            h, y = dev.download(H, (T, F), np.uint16), dev.download(Y, (T, D), np.uint16)
            up.check(x, starts, h)
            down.check(h, starts, y)
            up.plan.launch(up.args(X, s, H, ws[0]))
            down.plan.launch(down.args(H, s, Y, ws[1]))
            dev.sync()
            assert np.array_equal(dev.download(H, (T, F), np.uint16), h) and np.array_equal(dev.download(Y, (T, D), np.uint16), y)
    finally:
        for g in graphs:
            g.close()
    free(X, H, Y, s, *ws)
    up.close()
    down.close()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2000])  # few rows a workgroup, and large tiles
def test_every_scale(dev, dtype, N):
    # rows that somebody else has brought into the format: every scale byte, 0 (2^-127) among them, with every code
    R, K = 256 if N == 1 else 4096, 256
    codes = np.tile(np.arange(16, dtype=np.uint8) | (np.arange(16, dtype=np.uint8)[::-1] << 4), (R, 8))
    scales = np.repeat((np.arange(R) % 256).astype(np.uint8)[None, :, None], 8, 2)
    v = experts.values(codes, scales, K)
    d = [dev.upload(x) for x in (codes, np.ascontiguousarray(scales))]
    back = dev.upload(np.full((R, K), FILL, np.uint16))
    mtk.MxDequantizePlan(dev, R, K, dtype=dtype).run(*d, back)
    dev.sync()
    with np.errstate(over="ignore"):  # the largest are infinities in 16 bits
        want = kv.to_f64(kv.bits_of(v, dtype), dtype)
    got = kv.to_f64(dev.download(back, (R, K), np.uint16), dtype)
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]
    # times ones: the sum of each row's values; bf16 holds them all
    if dtype == "bf16":
        pick = np.r_[0:8]  # of a row, so that its sum is not zero
        ones = np.zeros((N, K))
        ones[:, pick] = 1
        qw = experts.quantise(kv.bits_of(ones, dtype), dtype)
        dw, out = [dev.upload(x) for x in qw], dev.empty(2 * R * N)
        plan = mtk.MxGemmPlan(dev, R, N, K, dtype=dtype)
        print(plan.describe(), flush=True)
        plan.run(*d, *dw, None, None, out)
        dev.sync()
        got = kv.to_f64(dev.download(out, (R, N), np.uint16), dtype)
        want, bound, _ = experts.mx_product(v, experts.values(*qw, K)[None], None, [0, R], dtype)
        nan, large = np.isnan(want), np.abs(want) > 2.0 ** 127  # (past the type, or near it)
        assert np.array_equal(np.isnan(got), nan)
        agree(got[~nan & ~large], want[~nan & ~large], bound[~nan & ~large], "C")
        free(out, *dw)
    free(back, *d)


# ------------------------------------------------------------------ streams, captures, several runs at once

def test_other_streams_and_captures(dev):
    E, T, N, K, dtype = 5, 900, 520, 640, "bf16"
    rng = rng_of(70)
    held = Held(dev, E, T, N, K, dtype, 71)
    assert held.plan.workspace_bytes
    A, dC, W = bits(rng, (T, K), dtype), bits(rng, (T, N), dtype), bits(rng, (E, N, K), dtype)
    d = [dev.upload(x) for x in (A, dC, W, routing(rng, T, E))]
    forward = mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype)
    grad = mtk.GroupedGradPlan(dev, E, T, N, K, dtype=dtype, has_bias=True)
    sizes = (2 * T * N, 2 * E * N * K, 2 * E * N, 2 * T * N, held.plan.workspace_bytes)  # C, dB, dbias, the product in 4 bits, its workspace
    outs = [[dev.empty(n) for n in sizes] for _ in range(3)]

    def run(o, ws):
        forward.run(d[0], d[2], None, d[3], o[0])
        grad.run(d[0], d[1], d[3], o[1], o[2])
        held.plan.launch(held.args(d[0], d[3], o[3], ws))

    def poison():
        for o in outs[:2]:
            for b in o:
                dev.upload_into(b, np.full(b.nbytes, 0xFF, np.uint8))

    for b in outs[2]:
        dev.upload_into(b, np.full(b.nbytes, 0xFF, np.uint8))
    run(outs[2], outs[2][4])
    dev.sync()
    want = [dev.download(b, (b.nbytes,), np.uint8) for b in outs[2][:4]]
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    streams = [ctypes.c_void_p() for _ in range(2)]
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()

    def same():
        assert hip.hipDeviceSynchronize() == 0
        for o in outs[:2]:
            for b, w in zip(o, want):
                assert np.array_equal(dev.download(b, w.shape, np.uint8), w)

    try:
        for s in streams:
            assert hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0  # non-blocking
        for _ in range(3):  # two runs at once, each with its own workspace
            poison()
            dev.sync()
            for s, o in zip(streams, outs):
                mtk._check(mtk.lib().mtk_set_stream(dev.handle, s))
                run(o, o[4])
            same()
        # two runs in one caller's capture that share a workspace: one after the other on one stream
        mtk._check(mtk.lib().mtk_set_stream(dev.handle, streams[0]))
        assert hip.hipStreamBeginCapture(streams[0], 2) == 0  # relaxed
        for o in outs[:2]:
            run(o, outs[0][4])
        assert hip.hipStreamEndCapture(streams[0], ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(3):
            poison()
            dev.sync()
            assert hip.hipGraphLaunch(graph_exec, streams[0]) == 0
            same()
    finally:
        mtk._check(mtk.lib().mtk_set_stream(dev.handle, None))
        for destroy, x in [("hipGraphExecDestroy", graph_exec), ("hipGraphDestroy", graph)] + [("hipStreamDestroy", s) for s in streams]:
            if x:
                getattr(hip, destroy)(x)
    free(*d, *[b for o in outs for b in o])
    held.close()


def test_profile(dev):
    E, T, N, K = 5, 900, 520, 640
    held = Held(dev, E, T, N, K, "f16", 72)
    rng = rng_of(73)
    A, dC, W, s = (dev.upload(x) for x in (bits(rng, (T, K), "f16"), bits(rng, (T, N), "f16"), bits(rng, (E, N, K), "f16"), routing(rng, T, E)))
    outs = [dev.empty(n) for n in (2 * T * N, 4 * E * N * K, 4 * E * N, max(16, held.plan.workspace_bytes))]
    forward = mtk.GroupedGemmPlan(dev, E, T, N, K)
    grad = mtk.GroupedGradPlan(dev, E, T, N, K, has_bias=True, out_f32=True)
    codes, scales = (dev.empty(n) for n in mtk.mx_bytes(T, K))
    there, back = mtk.MxQuantizePlan(dev, T, K), mtk.MxDequantizePlan(dev, T, K)
    for plan, args in ((forward, forward.args(A, W, None, s, outs[0])), (grad, grad.args(A, dC, s, outs[1], outs[2])),
                       (held.plan, held.args(A, s, outs[0], outs[3])), (there, there.args(A, codes, scales)), (back, back.args(codes, scales, A))):
        t = plan.profile([args], warmup=1, iters=3)
        print(t, flush=True)
        assert t["total_ms"] > 0 and len(t["kernels"]) == len(plan.describe().split("kernels: ")[1].split())
        flops, nbytes = plan.work()
        assert flops >= 0 and nbytes > 0
    free(A, dC, W, s, codes, scales, *outs)
    held.close()


# ------------------------------------------------------------------ past 2^32 bytes

def part(dev, buf, at, host):
    """A piece of a buffer, `at` bytes behind its start, with host's data in it."""
    piece = mtk.DeviceBuffer(dev, buf.ptr + at, host.nbytes)
    dev.upload_into(piece, host)
    return piece


@pytest.mark.parametrize("T", [24, 1500])  # a kernel for few rows, and large tiles
def test_weights_past_32_bits(dev, T):
    # only the first and the last weights of the last group hold anything; the outputs of those are compared
    E, N, K, dtype, n = 40, 14336, 4096, "bf16", 8
    rng, rows, cols = rng_of(80), np.r_[0:4, T - 4:T], np.r_[0:8, 14336 - 8:14336]
    B = dev.empty(2 * E * N * K)
    assert B.nbytes > 1 << 32
    A, w = bits(rng, (T, K), dtype), bits(rng, (2 * n, K), dtype, K ** -0.5)
    part(dev, B, 2 * (E - 1) * N * K, w[:n])
    part(dev, B, 2 * (E * N - n) * K, w[n:])
    dA, ds, dC = dev.upload(A), dev.upload(i32([0] * E + [T])), dev.upload(np.full((T, N), FILL, np.uint16))
    plan = mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype)
    print(plan.describe(), flush=True)
    plan.run(dA, B, None, ds, dC)
    dev.sync()
    got = dev.download(dC, (T, N), np.uint16)
    want, bound, _ = experts.grouped(A[rows], w[None], None, [0, 8], True, dtype)
    agree(kv.to_f64(got[np.ix_(rows, cols)], dtype), want, bound, "C")
    # in 4 bits, twice as many groups of rows of twice the length
    E, K = 2 * E, 2 * K
    A, w = bits(rng, (T, K), dtype), bits(rng, (2 * n, K), dtype, K ** -0.5)
    c, s = experts.quantise(w, dtype)
    codes, scales = mtk.mx_bytes(E * N, K)
    assert 1 << 32 < codes <= B.nbytes
    S = dev.empty(scales)
    for i, row in ((0, (E - 1) * N), (n, E * N - n)):
        part(dev, B, row * c.shape[1], c[i:i + n])
        for k in range(s.shape[0]):
            part(dev, S, (k * E * N + row) * 8, s[k, i:i + n])
    plan = mtk.MxGemmPlan(dev, T, N, K, E=E, dtype=dtype, quantize_a=True)
    print(plan.describe(), flush=True)
    dA2, ds2, ws = dev.upload(A), dev.upload(i32([0] * E + [T])), dev.empty(max(16, plan.workspace_bytes))
    plan.run(dA2, None, B, S, None, ds2, dC, ws)
    dev.sync()
    got = dev.download(dC, (T, N), np.uint16)
    v = experts.values(*experts.quantise(A[rows], dtype), K)
    want, bound, _ = experts.mx_product(v, experts.values(c, s, K)[None], None, [0, 8], dtype)
    agree(kv.to_f64(got[np.ix_(rows, cols)], dtype), want, bound, "C in 4 bits")
    free(B, S, dA, ds, dC, dA2, ds2, ws)


@pytest.mark.parametrize("E", [3, 14000])
def test_rows_past_32_bits(dev, E):
    T, N, K, dtype, n = (1 << 20) + 77, 2304, 64, "f16", 90
    rng = rng_of(81)
    A, B, C = dev.empty(2 * T * K), dev.empty(2 * E * N * K), dev.empty(2 * T * N)
    assert C.nbytes > 1 << 32
    dev.fill_u16(C, FILL, T * N)
    x, w = bits(rng, (n, K), dtype), bits(rng, (2, N, K), dtype)  # the last rows, of the last two groups
    part(dev, A, 2 * (T - n) * K, x)
    part(dev, B, 2 * (E - 2) * N * K, w)
    starts = np.full(E + 1, T - n)
    starts[E - 1], starts[E] = T - 40, T - 1
    plan = mtk.GroupedGemmPlan(dev, E, T, N, K, dtype=dtype)
    print(plan.describe(), flush=True)
    ds = dev.upload(i32(starts))
    plan.run(A, B, None, ds, C)
    dev.sync()
    rows = dev.download(mtk.DeviceBuffer(dev, C.ptr + 2 * (T - n - 5) * N, 2 * (n + 5) * N), (n + 5, N), np.uint16)
    want, bound, mine = experts.grouped(x, w, None, [0, n - 40, n - 1], True, dtype)
    assert (rows[:5] == FILL).all() and (rows[-1] == FILL).all()
    agree(kv.to_f64(rows[5:], dtype)[mine], want[mine], bound[mine], "C")
    free(A, B, C, ds)


def test_rows_in_4_bits_past_32_bits(dev):
    T, N, K, dtype, n = (1 << 20) + 77, 48, 8400, "bf16", 50
    rng = rng_of(83)
    src = dev.empty(2 * T * K)  # 17 GB
    dev.fill_u16(src, 0x3F80, T * K)  # ones
    x = bits(rng, (n, K), dtype)
    part(dev, src, 2 * (T - n) * K, x)
    codes, scales = (dev.empty(b) for b in mtk.mx_bytes(T, K))
    assert codes.nbytes > 1 << 32
    mtk.MxQuantizePlan(dev, T, K, dtype=dtype).run(src, codes, scales)
    dev.fill_u16(src, FILL, T * K)
    mtk.MxDequantizePlan(dev, T, K, dtype=dtype).run(codes, scales, src)
    W = bits(rng, (N, K), dtype, K ** -0.5)
    qw, q = experts.quantise(W, dtype), experts.quantise(x, dtype)
    dw, out = [dev.upload(b) for b in qw], dev.empty(2 * T * N)
    plan = mtk.MxGemmPlan(dev, T, N, K, dtype=dtype)
    print(plan.describe(), flush=True)
    plan.run(codes, scales, *dw, None, None, out)
    dev.sync()
    row = q[0].shape[1]
    assert np.array_equal(dev.download(mtk.DeviceBuffer(dev, codes.ptr + (T - n) * row, n * row), q[0].shape, np.uint8), q[0])
    v = experts.values(*q, K)
    back = dev.download(mtk.DeviceBuffer(dev, src.ptr + 2 * (T - n - 1) * K, 2 * (n + 1) * K), (n + 1, K), np.uint16)
    assert np.array_equal(kv.to_f64(back[1:], dtype), v) and (back[0] == 0x3F80).all()
    got = dev.download(mtk.DeviceBuffer(dev, out.ptr + 2 * (T - n) * N, 2 * n * N), (n, N), np.uint16)
    want, bound, _ = experts.mx_product(v, experts.values(*qw, K)[None], None, [0, n], dtype)
    agree(kv.to_f64(got, dtype), want, bound, "C")
    free(src, codes, scales, out, *dw)


@pytest.mark.parametrize("rows, out_f32", [(3, False), (900, False), (3, True), (900, True)])
def test_gradients_past_32_bits(dev, rows, out_f32):
    E, N, K, dtype = 140 >> out_f32, 4096, 4096, "bf16"
    rng = rng_of(82)
    T = rows
    A, dC = bits(rng, (T, K), dtype), bits(rng, (T, N), dtype)
    starts = i32([0] * E + [T])  # all rows are the last group's
    size = 4 if out_f32 else 2
    dB = dev.empty(size * E * N * K)
    assert dB.nbytes > 1 << 32
    dev.fill_u16(dB, FILL, dB.nbytes // 2)
    d = [dev.upload(x) for x in (A, dC, starts)]
    plan = mtk.GroupedGradPlan(dev, E, T, N, K, dtype=dtype, out_f32=out_f32)
    print(plan.describe(), flush=True)
    plan.run(*d, dB)
    dev.sync()
    kind = np.float32 if out_f32 else np.uint16
    last = dev.download(mtk.DeviceBuffer(dev, dB.ptr + size * (E - 1) * N * K, size * N * K), (N, K), kind)
    before = dev.download(mtk.DeviceBuffer(dev, dB.ptr + size * (E - 2) * N * K, size * N * K), (N, K), kind)
    assert not before.any()
    at = np.r_[0:40, N - 40:N]
    (want, bound), _ = experts.grad(A, np.ascontiguousarray(dC[:, at]), [0, T], True, dtype, "f32" if out_f32 else dtype)
    got = last[at].astype(np.float64) if out_f32 else kv.to_f64(last[at], dtype)
    agree(got, want[0], bound[0], "dB")
    free(dB, *d)
