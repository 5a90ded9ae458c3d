"""Work on a paged key/value cache held in few bits, as cases that can be timed and checked.

Three operators: `store` writes new rows of K and V into the cache (quantising them) and reads them back
in 16 bits, `fetch` reads a whole prefix back, `attend` is attention over the cache. With `own` false
`run` computes them in elementary torch operations in 32 bits, with `own` true through the library's plans.

The cache: n_pages pages of P positions; the region of (page, K/V head) holds K codes [P][row], V codes
[P][row], K scales [P][nb], V scales [P][nb], where a row is nb = ceil(D / 32) blocks of 32 dims (dims past D
are zeros) of 16 bytes (fp4: e2m1, two codes a byte, the even dim in the low half) or 32 bytes (fp8: e4m3),
and a scale byte s stands for 2^(s - 127); 255 makes its block NaN.
"""
import math
import random

import torch

own = False

_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # e2m1 magnitudes
_DEVICE = None


# ------------------------------------------------------------------ the cases


def _attend(name, lens, rows, H, H_kv, D, page, fmt="fp4", dtype="bf16", lse=False):
    """`lens`: "count x most / least", lengths spread over [least, most]; `rows`: new rows per sequence, or
    "first+others" where the first sequence has more than the others."""
    c = {"op": "attend", "lens": lens, "rows": rows, "H": H, "H_kv": H_kv, "D": D, "page": page, "fmt": fmt,
         "dtype": dtype, "lse": lse, "fused": False}
    return {"name": name, **c} if name else c


def _move(name, op, lens, rows, H, H_kv, D, page, fmt="fp4", dtype="bf16", fused=True):
    """`rows` "all": every position of the sequences."""
    c = {"op": op, "lens": lens, "rows": rows, "H": H, "H_kv": H_kv, "D": D, "page": page, "fmt": fmt, "dtype": dtype,
         "lse": False, "fused": fused}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's next token behind a short conversation: the call's latency is what is felt
        _attend("attend_1x1000", "1x1000/1000", "1+1", 32, 8, 128, 16),
        # a decode step of a serving batch with ragged lengths, grouped heads
        _attend("attend_32x4096", "32x4096/500", "1+1", 32, 8, 128, 64),
        # one token behind a very long document
        _attend("attend_1x131071", "1x131071/131071", "1+1", 32, 8, 128, 64, dtype="f16"),
        # a model with a K/V head for every query head, small head dimension, small pages
        _attend("attend_64x2048_mha", "64x2048/1500", "1+1", 16, 16, 64, 16, dtype="f16"),
        # the 8-bit cache, for users who want its accuracy
        _attend("attend_16x8192_fp8", "16x8192/6000", "1+1", 32, 8, 128, 32, fmt="fp8"),
        # five drafted tokens of each sequence checked at once
        _attend("attend_8x5_drafts", "8x8000/3000", "5+5", 32, 8, 128, 64),
        # a chunk of a prompt behind what is already cached; the row log-sum-exp lets a caller join it with other keys
        _attend("attend_chunk_2048", "1x8192/8192", "2048+1", 32, 8, 128, 64, lse=True),
        # a prompt's chunk and the other sequences' next tokens in one batch, 96-wide heads
        _attend("attend_mixed", "31x2000/700", "500+1", 24, 8, 96, 32, dtype="f16"),
        # a decode step's new rows: 64 tokens, one per sequence
        _move("store_64x1", "store", "64x4096/500", "1+1", 32, 8, 128, 64),
        # prompts as they come out of a fused projection
        _move("store_prompts", "store", "4x2500/1500", "all", 32, 8, 128, 64),
        # the 8-bit cache with 80-wide heads (a last block that is half empty), contiguous rows
        _move("store_fp8_d80", "store", "3x2100/1900", "all", 32, 32, 80, 16, fmt="fp8", dtype="f16", fused=False),
        # a cached prefix back to 16 bits, for a pass that wants it whole
        _move("fetch_32768", "fetch", "2x16384/16000", "all", 32, 8, 128, 64, fused=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of these ranges, no larger than the largest listed one."""
    while True:
        op = rng.choice(["attend", "attend", "attend", "attend", "store", "fetch"])
        H_kv = rng.choice([1, 2, 4, 8, 8, 16])
        H = H_kv * rng.choice([1, 1, 2, 4, 4, 7, 8])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 200, 256])
        B = _log(rng, 1, 64)
        most = _log(rng, 1, 131072 if op == "attend" else 16384)
        lens = "%dx%d/%d" % (B, most, max(1, int(most * rng.choice([1.0, 0.7, 0.1]))))
        page, fmt, dtype = rng.choice([16, 16, 32, 64, 128, 256]), rng.choice(["fp4", "fp4", "fp4", "fp8"]), rng.choice(["f16", "bf16"])
        if op == "attend":
            few = str(_log(rng, 2, 16))
            rows = rng.choice(["1+1", "1+1", "1+1", few + "+" + few, "%d+1" % _log(rng, 16, 2048), "%d+%d" % (_log(rng, 16, 2048), _log(rng, 1, 64))])
            c = _attend(None, lens, rows, H, H_kv, D, page, fmt, dtype, rng.random() < 0.3)
        else:
            c = _move(None, op, lens, "all" if op == "fetch" or rng.random() < 0.5 else "1+1", H, H_kv, D, page, fmt, dtype, rng.random() < 0.5)
        w = work(c)
        padded = B * max(_rows(c)) * H * most  # scores that the plain form holds at once
        if w["bytes"] <= 2.7e8 and w["flops"] <= 2.3e11 and padded <= 6e8:
            return c


# ------------------------------------------------------------------ inputs


def _lens(c):
    n, rest = c["lens"].split("x")
    most, least = (int(v) for v in rest.split("/"))
    r = random.Random(7 * int(n) + most)
    return [most if i == 0 else r.randint(least, most) for i in range(int(n))]


def _rows(c):
    lens = _lens(c)
    if c["rows"] == "all":
        return lens
    first, others = (int(v) for v in c["rows"].split("+"))
    return [min(lens[0], first)] + [min(n, others) for n in lens[1:]]


def _geometry(c):
    lens, P, nb = _lens(c), c["page"], (c["D"] + 31) // 32
    used = [(n + P - 1) // P for n in lens]
    row = nb * (16 if c["fmt"] == "fp4" else 32)
    return {"lens": lens, "rows": _rows(c), "B": len(lens), "T": sum(_rows(c)), "nb": nb, "row": row, "used": used,
            "max_pages": max(used), "n_pages": sum(used) + 3, "region": 2 * P * (row + nb)}


def _parts(c, cache):
    """(K codes, K scales, V codes, V scales), views [page][head][position][byte] of the cache."""
    g, P = _geometry(c), c["page"]
    at, out = 0, []
    for width in (g["row"], g["row"], g["nb"], g["nb"]):
        out.append(cache[:, :, at:at + P * width].unflatten(2, (P, width)))
        at += P * width
    return out[0], out[2], out[1], out[3]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _values(gen, n, c):
    """n rows of K and V: some dims of K are several times as large as others, as rotated keys have them."""
    shape = (n, c["H_kv"], c["D"])
    size = torch.exp(0.5 * torch.randn((1, c["H_kv"], c["D"]), generator=gen, device="cuda"))
    k = torch.randn(shape, generator=gen, device="cuda") * size
    v = torch.randn(shape, generator=gen, device="cuda")
    return k.to(_TORCH[c["dtype"]]), v.to(_TORCH[c["dtype"]])


def _inputs(c, seed):
    g, gen, P, dt = _geometry(c), _generator(seed), c["page"], _TORCH[c["dtype"]]
    order = torch.randperm(g["n_pages"], generator=gen, device="cuda").to(torch.int32)
    table = torch.full((g["B"], g["max_pages"]), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(g["used"]):  # the sequences' pages lie anywhere in the cache
        table[b, :n] = order[at:at + n]
        at += n
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    start = [0]
    for n in g["rows"]:
        start.append(start[-1] + n)
    t = {"table": table, "row_start": ints(start), "kv_len": ints(g["lens"])}
    cache = torch.zeros((g["n_pages"], c["H_kv"], g["region"]), dtype=torch.uint8, device="cuda")
    if c["op"] != "store":
        parts = _parts(c, cache)
        for p0 in range(0, g["n_pages"], max(1, 65536 // P)):
            n = min(g["n_pages"], p0 + max(1, 65536 // P)) - p0
            for i, x in enumerate(_values(gen, n * P, c)):
                codes, scales = _quantise(x, c["fmt"])
                parts[2 * i][p0:p0 + n] = codes.unflatten(0, (n, P)).transpose(1, 2)
                parts[2 * i + 1][p0:p0 + n] = scales.unflatten(0, (n, P)).transpose(1, 2)
    else:
        if c["fused"]:  # [row][query heads, K heads, V heads]
            t["qkv"] = torch.zeros((g["T"], c["H"] + 2 * c["H_kv"], c["D"]), dtype=dt, device="cuda")
            t["K"], t["V"] = t["qkv"][:, c["H"]:c["H"] + c["H_kv"]], t["qkv"][:, c["H"] + c["H_kv"]:]
            k, v = _values(gen, g["T"], c)
            t["K"].copy_(k)
            t["V"].copy_(v)
        else:
            t["K"], t["V"] = _values(gen, g["T"], c)
    t["cache"] = cache
    if c["op"] == "attend":
        t["Q"] = torch.randn((g["T"], c["H"], c["D"]), generator=gen, device="cuda").to(dt)
    return t


def prepare(case, seed):
    """What a program holds before the call: inputs and outputs on the GPU, the library's plans and their workspace."""
    c, t, g = case, _inputs(case, seed), _geometry(case)
    dt = _TORCH[c["dtype"]]
    if c["op"] == "attend":
        out = {"O": torch.empty_like(t["Q"])}
        if c["lse"]:
            out["lse"] = torch.empty((g["T"], c["H"]), dtype=torch.float32, device="cuda")
    else:
        out = {n: torch.empty((g["T"], c["H_kv"], c["D"]), dtype=dt, device="cuda") for n in "KV"}
    state = {"case": c, "in": t, "out": out}
    if own:
        state["steps"], state["keep"] = _plans(c, g, t, out)
    torch.cuda.synchronize()  # the inputs were made on torch's stream, the plans run on the library's
    return state


def _plans(c, g, t, out):
    global _DEVICE
    import example_matmul_metal4_amd as mtk
    if _DEVICE is None:
        _DEVICE = mtk.Device(0)
    p = lambda x: x.data_ptr()
    batch = (p(t["row_start"]), p(t["kv_len"]), p(t["table"]))
    pages = {"n_pages": g["n_pages"], "page_size": c["page"], "max_pages": g["max_pages"], "format": c["fmt"], "dtype": c["dtype"]}
    if c["op"] == "attend":
        plan = mtk.KvAttentionPlan(_DEVICE, g["B"], g["T"], c["H"], c["H_kv"], c["D"], S_q=max(g["rows"]), **pages)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda") if plan.workspace_bytes else None
        args = plan.args(p(t["Q"]), p(t["cache"]), *batch, p(out["O"]), p(out["lse"]) if c["lse"] else None,
                         None if ws is None else p(ws))
        return [(plan, args)], ws
    steps = []
    if c["op"] == "store":
        plan = mtk.KvWritePlan(_DEVICE, g["B"], g["T"], c["H_kv"], c["D"], ld_k=t["K"].stride(0), ld_v=t["V"].stride(0), **pages)
        steps.append((plan, plan.args(p(t["K"]), p(t["V"]), p(t["cache"]), *batch)))
    plan = mtk.KvReadPlan(_DEVICE, g["B"], g["T"], c["H_kv"], c["D"], **pages)
    steps.append((plan, plan.args(p(t["cache"]), *batch, p(out["K"]), p(out["V"]))))
    return steps, None


def run(state):
    if "steps" in state:
        for plan, args in state["steps"]:
            plan.launch(args)
        return state["out"]
    c, t = state["case"], state["in"]
    if c["op"] == "attend":
        return _attend_plain(c, t)
    if c["op"] == "store":
        _store_plain(c, t)
    return _fetch_plain(c, t)


# ------------------------------------------------------------------ the plain forms


def _quantise(x, fmt):
    """Rows [n][H_kv][D] in 16 bits -> codes [n][H_kv][nb * 16 or 32], scales [n][H_kv][nb], bytes."""
    limit = (1.5 if fmt == "fp4" else 1.875) * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    bad = (~torch.isfinite(x)).any(-1)
    x = torch.where(bad[..., None], 0.0, x).clamp(-limit, limit)
    m, k = torch.frexp(x.abs().amax(-1))  # amax = m 2^k with 0.5 <= m < 1
    if fmt == "fp4":
        e = torch.where(m <= 0.75, k - 3, k - 2)  # 6 = 0.75 * 2^3
    else:
        e = torch.where(m <= 0.875, k - 9, k - 8)  # 448 = 0.875 * 2^9
    e = torch.where(m > 0, e, -126).clamp(min=-126)
    a = torch.ldexp(x.abs(), -e[..., None])
    if fmt == "fp4":
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    else:
        step = torch.exp2(torch.frexp(a)[1].clamp(min=-5).float() - 4)  # 4 significant bits, at least 2^-9
    a = torch.round(a / step) * step
    if fmt == "fp4":
        code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).to(torch.int32)
    else:
        m, k = torch.frexp(a)
        code = torch.where(a < 2.0 ** -6, a * 512, (k + 6).float() * 8 + (m * 16 - 8)).to(torch.int32)
    code = code + torch.where(torch.signbit(x), 8 if fmt == "fp4" else 128, 0)
    code = code.flatten(-2)
    if fmt == "fp4":
        code = code[..., 0::2] + code[..., 1::2] * 16
    return code.to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def _dequantise(codes, scales, D):
    """The values of codes [..][nb * 16 or 32] with scales [..][nb], in 32 bits: [..][D]."""
    if codes.shape[-1] == 16 * scales.shape[-1]:
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        a = (n & 7).float()
        v = torch.where(a < 4, a * 0.5, torch.where(a < 6, a - 2, a * 2 - 8))
        v = torch.where(n >= 8, -v, v)
    else:
        a = (codes & 127).float()
        e, m = torch.floor(a / 8), a - 8 * torch.floor(a / 8)
        v = torch.where(e > 0, torch.exp2(e - 10) * (8 + m), m / 512)
        v = torch.where(codes >= 128, -v, v)
    s = scales.float()
    s = torch.where(s < 255, torch.exp2(s - 127), math.nan)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :D]


def _places(c, t, pos, b):
    """(page, offset) of positions `pos` of sequences `b`."""
    return t["table"][b, pos // c["page"]].long(), pos % c["page"]


def _new_rows(c, t):
    """(sequence, position) of each row of the packed tensors."""
    start, T = t["row_start"].long(), _geometry(c)["T"]
    i = torch.arange(T, device="cuda")
    b = torch.searchsorted(start, i, right=True) - 1
    return b, t["kv_len"].long()[b] - (start[b + 1] - i)


def _store_plain(c, t):
    b, pos = _new_rows(c, t)
    page, off = _places(c, t, pos, b)
    parts = _parts(c, t["cache"])
    for i, n in enumerate("KV"):
        codes, scales = _quantise(t[n], c["fmt"])
        parts[2 * i][page, :, off] = codes
        parts[2 * i + 1][page, :, off] = scales


def _fetch_plain(c, t):
    b, pos = _new_rows(c, t)
    page, off = _places(c, t, pos, b)
    kc, ks, vc, vs = _parts(c, t["cache"])
    dt = _TORCH[c["dtype"]]
    return {"K": _dequantise(kc[page, :, off], ks[page, :, off], c["D"]).to(dt),
            "V": _dequantise(vc[page, :, off], vs[page, :, off], c["D"]).to(dt)}


def _attend_plain(c, t):
    g = _geometry(c)
    B, L, S, H_kv, D = g["B"], max(g["lens"]), max(g["rows"]), c["H_kv"], c["D"]
    G = c["H"] // H_kv
    kv_len, start = t["kv_len"].long(), t["row_start"].long()
    pos = torch.arange(L, device="cuda")
    seq = torch.arange(B, device="cuda")[:, None]
    page, off = _places(c, t, pos[None].expand(B, L), seq)
    page = page.clamp(min=0)
    keys = []
    for codes, scales in (_parts(c, t["cache"])[:2], _parts(c, t["cache"])[2:]):
        x = _dequantise(codes[page, :, off], scales[page, :, off], D)  # [B][L][H_kv][D]
        keys.append(x.permute(0, 2, 1, 3).reshape(B * H_kv, L, D))
    inside = pos[None] < kv_len[:, None]
    k, v = keys[0], torch.where(inside[:, None, :, None], keys[1].view(B, H_kv, L, D), 0.0).view(B * H_kv, L, D)
    b, p = _new_rows(c, t)
    i = torch.arange(g["T"], device="cuda") - start[b]
    q = torch.zeros((B, S, H_kv, G, D), device="cuda")
    q[b, i] = t["Q"].float().view(-1, H_kv, G, D)
    at = torch.zeros((B, S), dtype=torch.long, device="cuda")
    at[b, i] = p
    q = q.permute(0, 2, 1, 3, 4).reshape(B * H_kv, S * G, D)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(B, H_kv, S, G, L) * (1 / math.sqrt(D))
    s = torch.where((pos[None, None] <= at[..., None])[:, None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - m)
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(B * H_kv, S * G, L), v).view(B, H_kv, S, G, D) / total
    pick = lambda x: x.permute(0, 2, 1, 3, 4)[b, i].flatten(1, 2)  # [T][H][..]
    out = {"O": pick(o).to(_TORCH[c["dtype"]])}
    if c["lse"]:
        out["lse"] = pick(m + torch.log(total))[..., 0]
    return out


# ------------------------------------------------------------------ work and 64-bit results


def work(case):
    c, g = case, _geometry(case)
    rows16 = 2 * g["T"] * c["H_kv"] * c["D"]  # bytes of the new rows of K, or of V
    per = 2 * c["H_kv"] * (g["row"] + g["nb"])  # bytes of a cached position
    ints = 4 * (2 * g["B"] + 1)
    if c["op"] == "attend":
        pairs = sum(n * (2 * (length - n) + n + 1) // 2 for n, length in zip(g["rows"], g["lens"]))
        q = 2 * g["T"] * c["H"] * c["D"]
        return {"bytes": per * sum(g["lens"]) + 2 * q + (4 * g["T"] * c["H"] if c["lse"] else 0) + ints + 4 * sum(g["used"]),
                "flops": 4 * c["H"] * c["D"] * pairs}
    if c["op"] == "store":
        return {"bytes": 4 * rows16 + per * g["T"] + ints, "flops": 0}
    return {"bytes": 2 * rows16 + per * g["T"] + ints, "flops": 0}


def _grid64(fmt):
    """Every magnitude of the format, ascending by code, in 64 bits."""
    if fmt == "fp4":
        g = _GRID
    else:
        g = [(n % 8) * 2.0 ** -9 if n < 8 else (8 + n % 8) * 2.0 ** (n // 8 - 10) for n in range(127)]
    return torch.tensor(g, dtype=torch.float64, device="cuda")


def _held(x, fmt):
    """What the cache holds for 16-bit rows x, in 64 bits: for each block of 32 the smallest power of two that brings
    its largest magnitude into the format's range, and the nearest value of the format, ties to the even code."""
    grid = _grid64(fmt)
    most = (1.5 if fmt == "fp4" else 1.875) * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    for d in range(0, x.shape[-1], 32):
        y = x[..., d:d + 32].double().clamp(-most, most)
        top = y.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / grid[-1]))
        e = torch.where(top > grid[-1] * torch.exp2(e), e + 1, e)
        e = torch.where(top <= grid[-1] * torch.exp2(e - 1), e - 1, e)
        one = torch.exp2(e.clamp(min=-126))
        a = y.abs() / one
        low = torch.searchsorted(mid, a.contiguous())  # ties fall on the lower code
        tie = (low < len(mid)) & (a == mid[low.clamp(max=len(mid) - 1)])
        low = torch.where(tie & (low % 2 == 1), low + 1, low)
        out[..., d:d + 32] = torch.where(y < 0, -grid[low], grid[low]) * one
    return out


def _cached64(c, cache, table, length, head, which):
    """K (0) or V (1) of one sequence and head in 64 bits, [length][D]."""
    g, P = _geometry(c), c["page"]
    n = (length + P - 1) // P
    region = cache[table[:n].long(), head]  # [page][bytes]
    code = region[:, which * P * g["row"]:(which + 1) * P * g["row"]].reshape(n * P, g["row"])[:length].long()
    at = 2 * P * g["row"] + which * P * g["nb"]
    scale = region[:, at:at + P * g["nb"]].reshape(n * P, g["nb"])[:length].double()
    grid = _grid64(c["fmt"])
    both = torch.cat([grid, -grid]) if c["fmt"] == "fp4" else torch.cat([grid, grid[:1] / 0, -grid, grid[:1] / 0])
    if c["fmt"] == "fp4":
        code = torch.stack((code % 16, code // 16), 2).reshape(length, -1)
    return both[code][:, :c["D"]] * torch.exp2(scale - 127).repeat_interleave(32, 1)[:, :c["D"]]


def exact(case, seed):
    c, g, t = case, _geometry(case), _inputs(case, seed)
    if c["op"] == "store":
        return {n: _held(t[n], c["fmt"]) for n in "KV"}
    first = [0]
    for n in g["rows"]:
        first.append(first[-1] + n)
    if c["op"] == "fetch":
        out = {n: torch.empty((g["T"], c["H_kv"], c["D"]), dtype=torch.float64, device="cuda") for n in "KV"}
        for b, n in enumerate(g["lens"]):
            for h in range(c["H_kv"]):
                for i, name in enumerate("KV"):
                    out[name][first[b]:first[b + 1], h] = _cached64(c, t["cache"], t["table"][b], n, h, i)[n - g["rows"][b]:]
        return out
    out = {"O": torch.empty(t["Q"].shape, dtype=torch.float64, device="cuda")}
    lse = torch.empty(t["Q"].shape[:2], dtype=torch.float64, device="cuda")
    G = c["H"] // c["H_kv"]
    for b, (n, length) in enumerate(zip(g["rows"], g["lens"])):
        j = torch.arange(length, device="cuda")
        for h in range(c["H"]):
            if h % G == 0:
                k, v = (_cached64(c, t["cache"], t["table"][b], length, h // G, i) for i in (0, 1))
                kt = k.t().contiguous()
            q = t["Q"][first[b]:first[b + 1], h].double()
            s = (q @ kt) / math.sqrt(c["D"])
            i = torch.arange(n, device="cuda") + (length - n)
            s = s.masked_fill(j[None] > i[:, None], -math.inf)
            z = torch.logsumexp(s, 1, keepdim=True)
            out["O"][first[b]:first[b + 1], h] = torch.exp(s - z) @ v
            lse[first[b]:first[b + 1], h] = z[:, 0]
    if c["lse"]:
        out["lse"] = lse
    return out
