"""Products of a mixture of experts' layers and of layers held in 4 bits, as cases that can be timed and checked.

Four operators. `grouped`: rows sorted by expert times each expert's weights, C[t] = A[t] op(B_e) + bias_e for the rows
t of expert e (with `trans_b` false it is the input gradient of the same layer). `grad`: the gradients of the weights and of
the bias, dB_e = dC_e^T A_e and the column sums of dC_e. `rows`: 16-bit rows into blocks of 32 four-bit values with one
power-of-two scale, and back. `mx`: the product of 16-bit rows, brought into that format, with weights held in it, whole or
grouped by expert. With `own` false `run` computes them in elementary torch operations in 32 bits, with `own` true through
the library's plans.

Rows in few bits: K is padded with zeros to a multiple of 256. Codes [R][K / 2] (e2m1, two a byte, the even place in the low
half), scales [K / 256][R][8]: a byte s stands for 2^(s - 127); 255 makes its block of 32 NaN.
"""
import math
import random

import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # e2m1 magnitudes
_DEVICE = None


# ------------------------------------------------------------------ the cases


def _case(name, op, T, E, N, K, skew=0.0, dtype="bf16", trans_b=True, bias=False, out="16"):
    """`skew`: expert i is chosen in proportion to 1 / (1 + i)^skew. E 0: one product of all rows. `out` "f32": gradients
    in 32 bits. N and `trans_b` say nothing to `rows`, which has T rows of K values."""
    c = {"op": op, "T": T, "E": E, "N": N, "K": K, "skew": skew, "dtype": dtype, "trans_b": trans_b, "bias": bias, "out": out}
    return {"name": name, **c} if name else c


def listed():
    return [
        # eight users' next tokens, two experts each: the weights of a few experts are read for a row or two
        _case("grouped_16", "grouped", 16, 32, 2048, 2048, 0.5),
        # a serving batch's step over few wide experts: all weights are read, for about 30 rows each
        _case("grouped_256", "grouped", 256, 8, 14336, 4096, 0.3),
        # prompts, or the forward pass of a training step
        _case("grouped_8192", "grouped", 8192, 16, 4096, 4096, 0.3, "f16", bias=True),
        # the input gradient of such a layer with many small experts, some of them much busier than others
        _case("grouped_dx_8192", "grouped", 8192, 64, 1536, 2048, 0.8, trans_b=False),
        # odd sizes throughout
        _case("grouped_odd_1023", "grouped", 1023, 7, 1001, 1023, 0.5, "f16", bias=True),
        # the weights' gradients of the training step
        _case("grad_8192", "grad", 8192, 16, 4096, 4096, 0.3),
        # a small step's, kept in 32 bits, experts without any row among them
        _case("grad_1000", "grad", 1000, 24, 1023, 520, 1.2, "f16", bias=True, out="f32"),
        # one batch of next tokens into 4 bits and back
        _case("rows_16x4096", "rows", 16, 0, 0, 4096),
        # a prompt's rows, of a width that is no whole number of blocks
        _case("rows_8192x4100", "rows", 8192, 0, 0, 4100, dtype="f16"),
        # next tokens through a wide layer held in 4 bits
        _case("mx_16x14336", "mx", 16, 0, 14336, 4096),
        # a prompt through it
        _case("mx_4096x14336", "mx", 4096, 0, 14336, 4096, bias=True),
        # prompts through experts held in 4 bits
        _case("mx_grouped_8192", "mx", 8192, 32, 2048, 2048, 0.5, "f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A layer's width: a multiple of 64 mostly, of 8, or any."""
    return max(1, _log(rng, lo, hi) // (step := rng.choice([64, 64, 64, 8, 1])) * step)


def draw(rng):
    """One more case of these ranges, no larger than the largest listed one."""
    while True:
        op = rng.choice(["grouped", "grouped", "grouped", "grad", "grad", "rows", "mx", "mx", "mx"])
        T = _log(rng, 1, 16384)
        E = rng.choice([1, 2, 4, 7, 8, 16, 32, 64, 100, 128])
        N, K = _size(rng, 64, 14336), _size(rng, 64, 14336)
        skew, dtype = rng.choice([0.0, 0.3, 0.5, 0.8, 1.2]), rng.choice(["f16", "bf16"])
        bias = rng.random() < 0.4
        if op == "grouped":
            c = _case(None, op, T, E, N, K, skew, dtype, rng.random() < 0.6, bias)
        elif op == "grad":
            c = _case(None, op, T, E, N, K, skew, dtype, rng.random() < 0.6, bias, rng.choice(["16", "f32"]))
        elif op == "rows":
            c = _case(None, op, T, 0, 0, K, 0.0, dtype)
        else:
            c = _case(None, op, T, rng.choice([0, 0, E]), N, K, skew, dtype, True, bias)
        w = work(c)
        if w["bytes"] <= 1e9 and w["flops"] <= 2.8e11 and max(E, 1) * N * K <= 5e8:
            return c


# ------------------------------------------------------------------ inputs


def _starts(c):
    """Where each expert's rows start, and the end."""
    E, T = max(1, c["E"]), c["T"]
    r = random.Random(1000 * E + T)
    weights = [1.0 / (1 + i) ** c["skew"] for i in range(E)]
    r.shuffle(weights)
    count = [0] * E
    for e in r.choices(range(E), weights, k=T):
        count[e] += 1
    start = [0]
    for n in count:
        start.append(start[-1] + n)
    return start


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _padded(K):
    return -(-K // 256) * 256


def _activations(gen, T, K, dt):
    """Rows whose places are of different sizes, some few of them ten times as large."""
    size = torch.exp(0.5 * torch.randn((1, K), generator=gen, device="cuda"))
    size = torch.where(torch.rand((1, K), generator=gen, device="cuda") < 0.01, 10 * size, size)
    return (torch.randn((T, K), generator=gen, device="cuda") * size).to(dt)


def _inputs(c, seed):
    gen, dt = _generator(seed), _TORCH[c["dtype"]]
    E, T, N, K = max(1, c["E"]), c["T"], c["N"], c["K"]
    t = {}
    if c["op"] in ("rows", "mx"):
        t["A"] = _activations(gen, T, K, dt)
    else:
        t["A"] = torch.randn((T, K), generator=gen, device="cuda").to(dt)
    t["row_start"] = torch.tensor(_starts(c), dtype=torch.int32, device="cuda")
    if c["op"] == "grad":
        t["dC"] = torch.randn((T, N), generator=gen, device="cuda").to(dt)
    if c["op"] == "grouped":
        t["B"] = torch.empty((E, N, K) if c["trans_b"] else (E, K, N), dtype=dt, device="cuda")
        for e in range(E):
            t["B"][e] = torch.randn(t["B"].shape[1:], generator=gen, device="cuda") * (1 / math.sqrt(K))
    if c["op"] == "mx":
        Kp = _padded(K)
        t["codes"] = torch.empty((E * N, Kp // 2), dtype=torch.uint8, device="cuda")
        t["scales"] = torch.empty((Kp // 256, E * N, 8), dtype=torch.uint8, device="cuda")
        for e in range(E):
            w = (torch.randn((N, K), generator=gen, device="cuda") * (1 / math.sqrt(K))).to(dt)
            t["codes"][e * N:(e + 1) * N], t["scales"][:, e * N:(e + 1) * N] = _quantise(w)
    if c["bias"] and c["op"] != "grad":
        t["bias"] = torch.randn((E, N), generator=gen, device="cuda").to(dt)
    return t


def prepare(case, seed):
    """What a program holds before the call: inputs and outputs on the GPU, the library's plans and their workspace."""
    c, t = case, _inputs(case, seed)
    E, T, N, K, dt = max(1, c["E"]), c["T"], c["N"], c["K"], _TORCH[c["dtype"]]
    empty = lambda shape, kind: torch.empty(shape, dtype=kind, device="cuda")
    if c["op"] == "grad":
        kind = torch.float32 if c["out"] == "f32" else dt
        out = {"dB": empty((E, N, K) if c["trans_b"] else (E, K, N), kind)}
        if c["bias"]:
            out["dbias"] = empty((E, N), kind)
    elif c["op"] == "rows":
        out = {"values": empty((T, K), dt)}
    else:
        out = {"C": empty((T, N), dt)}
    state = {"case": c, "in": t, "out": out, "starts": _starts(c)}
    if own:
        state["steps"], state["keep"] = _plans(c, t, out)
    torch.cuda.synchronize()  # the inputs were made on torch's stream, the plans run on the library's
    return state


def _plans(c, t, out):
    global _DEVICE
    import example_matmul_metal4_amd as mtk
    if _DEVICE is None:
        _DEVICE = mtk.Device(0)
    p = lambda x: None if x is None else x.data_ptr()
    space = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    E, T, N, K = c["E"], c["T"], c["N"], c["K"]
    if c["op"] == "rows":
        codes, scales = (space(n) for n in mtk.mx_bytes(T, K))
        write = mtk.MxQuantizePlan(_DEVICE, T, K, dtype=c["dtype"])
        read = mtk.MxDequantizePlan(_DEVICE, T, K, dtype=c["dtype"])
        return [(write, write.args(p(t["A"]), p(codes), p(scales))),
                (read, read.args(p(codes), p(scales), p(out["values"])))], (codes, scales)
    if c["op"] == "grouped":
        plan = mtk.GroupedGemmPlan(_DEVICE, E, T, N, K, trans_b=c["trans_b"], dtype=c["dtype"], has_bias=c["bias"])
        ws = space(plan.workspace_bytes)
        return [(plan, plan.args(p(t["A"]), p(t["B"]), p(t.get("bias")), p(t["row_start"]), p(out["C"]), p(ws)))], ws
    if c["op"] == "grad":
        plan = mtk.GroupedGradPlan(_DEVICE, E, T, N, K, trans_b=c["trans_b"], dtype=c["dtype"], has_bias=c["bias"],
                                   out_f32=c["out"] == "f32")
        ws = space(plan.workspace_bytes)
        return [(plan, plan.args(p(t["A"]), p(t["dC"]), p(t["row_start"]), p(out["dB"]), p(out.get("dbias")), p(ws)))], ws
    plan = mtk.MxGemmPlan(_DEVICE, T, N, K, E=E, dtype=c["dtype"], has_bias=c["bias"], quantize_a=True)
    ws = space(plan.workspace_bytes)
    return [(plan, plan.args(p(t["A"]), None, p(t["codes"]), p(t["scales"]), p(t.get("bias")), p(t["row_start"]) if E else None,
                             p(out["C"]), p(ws)))], ws


def run(state):
    if "steps" in state:
        for plan, args in state["steps"]:
            plan.launch(args)
        return state["out"]
    c, t, start = state["case"], state["in"], state["starts"]
    return {"grouped": _grouped_plain, "grad": _grad_plain, "rows": _rows_plain, "mx": _mx_plain}[c["op"]](c, t, start)


# ------------------------------------------------------------------ the plain forms


def _quantise(x):
    """Rows [R][K] in 16 bits -> codes [R][Kp / 2], scales [Kp / 256][R][8], bytes."""
    limit = 1.5 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    R, K = x.shape
    x = torch.nn.functional.pad(x.float(), (0, _padded(K) - K)).unflatten(-1, (-1, 32))
    bad = (~torch.isfinite(x)).any(-1)
    x = torch.where(bad[..., None], 0.0, x).clamp(-limit, limit)
    m, k = torch.frexp(x.abs().amax(-1))  # amax = m 2^k with 0.5 <= m < 1
    e = torch.where(m <= 0.75, k - 3, k - 2)  # 6 = 0.75 * 2^3
    e = torch.where(m > 0, e, -126).clamp(min=-126)
    a = torch.ldexp(x.abs(), -e[..., None])
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).to(torch.int32)
    code = (code + torch.where(torch.signbit(x), 8, 0)).flatten(-2)
    code = code[..., 0::2] + code[..., 1::2] * 16
    scale = torch.where(bad, 255, e + 127).to(torch.uint8)
    return code.to(torch.uint8), scale.unflatten(1, (-1, 8)).transpose(0, 1).contiguous()


def _dequantise(codes, scales, K):
    """The values of codes [R][Kp / 2] with scales [Kp / 256][R][8], in 32 bits: [R][K]."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    a = (n & 7).float()
    v = torch.where(a < 4, a * 0.5, torch.where(a < 6, a - 2, a * 2 - 8))
    v = torch.where(n >= 8, -v, v)
    s = scales.transpose(0, 1).flatten(1).float()
    s = torch.where(s < 255, torch.exp2(s - 127), math.nan)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :K]


def _busy(start):
    return [(e, start[e], start[e + 1]) for e in range(len(start) - 1) if start[e + 1] > start[e]]


def _grouped_plain(c, t, start):
    out = torch.empty((c["T"], c["N"]), dtype=_TORCH[c["dtype"]], device="cuda")
    for e, i, j in _busy(start):
        w = t["B"][e].float()
        x = t["A"][i:j].float() @ (w.t() if c["trans_b"] else w)
        if c["bias"]:
            x = x + t["bias"][e].float()
        out[i:j] = x
    return {"C": out}


def _grad_plain(c, t, start):
    E, N, K = c["E"], c["N"], c["K"]
    kind = _TORCH["f32" if c["out"] == "f32" else c["dtype"]]
    out = {"dB": torch.zeros((E, N, K) if c["trans_b"] else (E, K, N), dtype=kind, device="cuda")}
    if c["bias"]:
        out["dbias"] = torch.zeros((E, N), dtype=kind, device="cuda")
    for e, i, j in _busy(start):
        a, d = t["A"][i:j].float(), t["dC"][i:j].float()
        out["dB"][e] = d.t() @ a if c["trans_b"] else a.t() @ d
        if c["bias"]:
            out["dbias"][e] = d.sum(0)
    return out


def _rows_plain(c, t, start):
    return {"values": _dequantise(*_quantise(t["A"]), c["K"]).to(_TORCH[c["dtype"]])}


def _mx_plain(c, t, start):
    N, K = c["N"], c["K"]
    a = _dequantise(*_quantise(t["A"]), K)
    out = torch.empty((c["T"], N), dtype=_TORCH[c["dtype"]], device="cuda")
    for e, i, j in _busy(start):
        x = a[i:j] @ _dequantise(t["codes"][e * N:(e + 1) * N], t["scales"][:, e * N:(e + 1) * N], K).t()
        if c["bias"]:
            x = x + t["bias"][e].float()
        out[i:j] = x
    return {"C": out}


# ------------------------------------------------------------------ work and 64-bit results


def work(case):
    c = case
    T, E, N, K = c["T"], max(1, c["E"]), c["N"], c["K"]
    start = _starts(c)
    busy = len(_busy(start))  # the weights of experts without a row need not be read
    ints = 4 * (E + 1) if c["E"] else 0
    if c["op"] == "rows":
        per = _padded(K) // 2 + _padded(K) // 32
        return {"bytes": T * (4 * K + 2 * per), "flops": 0}
    if c["op"] == "grad":
        size = 4 if c["out"] == "f32" else 2
        return {"bytes": 2 * T * (N + K) + size * E * N * (K + (1 if c["bias"] else 0)) + ints, "flops": 2 * T * N * K}
    rows = 2 * T * (N + K) + (2 * busy * N if c["bias"] else 0) + ints
    if c["op"] == "grouped":
        return {"bytes": rows + 2 * busy * N * K, "flops": 2 * T * N * K}
    return {"bytes": rows + busy * N * (_padded(K) // 2 + _padded(K) // 32), "flops": 2 * T * N * K}


def _held64(x):
    """What 16-bit rows x become, in 64 bits: for each block of 32 the smallest power of two that brings its largest
    magnitude to at most 6, and the nearest e2m1 value, ties to the even code."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device="cuda")
    mid = (grid[1:] + grid[:-1]) / 2
    most = 1.5 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for d in range(0, x.shape[1], 32):
        y = x[:, d:d + 32].double().clamp(-most, most)
        top = y.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6))
        e = torch.where(top > 6 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 6 * torch.exp2(e - 1), e - 1, e)
        one = torch.exp2(e.clamp(min=-126))
        a = y.abs() / one
        low = torch.searchsorted(mid, a.contiguous())  # ties fall on the lower code
        tie = (low < 7) & (a == mid[low.clamp(max=6)])
        low = torch.where(tie & (low % 2 == 1), low + 1, low)
        out[:, d:d + 32] = torch.where(y < 0, -grid[low], grid[low]) * one
    return out


def _weights64(c, t, e):
    """Expert e's weights held in few bits, in 64 bits: [N][K]."""
    N, K = c["N"], c["K"]
    grid = torch.tensor(_GRID + [-v for v in _GRID], dtype=torch.float64, device="cuda")
    code = t["codes"][e * N:(e + 1) * N].long()
    scale = torch.exp2(t["scales"][:, e * N:(e + 1) * N].double() - 127)  # [Kp / 256][N][8]
    w = torch.empty((N, _padded(K)), dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = grid[code % 16], grid[code // 16]
    for k in range(0, _padded(K), 32):
        w[:, k:k + 32] *= scale[k // 256, :, k % 256 // 32, None]
    return w[:, :K].contiguous()


def exact(case, seed):
    c, t, start = case, _inputs(case, seed), _starts(case)
    E, T, N, K = max(1, c["E"]), c["T"], c["N"], c["K"]
    zeros = lambda shape: torch.zeros(shape, dtype=torch.float64, device="cuda")
    if c["op"] == "rows":
        return {"values": _held64(t["A"])}
    if c["op"] == "grad":
        out = {"dB": zeros((E, N, K))}
        if c["bias"]:
            out["dbias"] = zeros((E, N))
        for e in range(E):
            d = t["dC"][start[e]:start[e + 1]].double()
            out["dB"][e] = torch.mm(d.t().contiguous(), t["A"][start[e]:start[e + 1]].double())
            if c["bias"]:
                out["dbias"][e] = d.sum(0)
        if not c["trans_b"]:
            out["dB"] = out["dB"].transpose(1, 2).contiguous()
        return out
    out = zeros((T, N))
    a = _held64(t["A"]) if c["op"] == "mx" else t["A"].double()
    for e in range(E):
        i, j = start[e], start[e + 1]
        if i == j:
            continue
        if c["op"] == "mx":
            w = _weights64(c, t, e).t().contiguous()
        else:
            w = t["B"][e].double()
            w = w.t().contiguous() if c["trans_b"] else w
        out[i:j] = torch.mm(a[i:j], w)
        if c["bias"]:
            out[i:j] += t["bias"][e].double()
    return {"C": out}
