"""The paged key/value cache in few bits (include/mtk.h) in numpy and 64 bits: the plain implementation that the
tests compare with. f16 tensors are numpy float16, bf16 tensors uint16 bit patterns, as in the rest of the package."""
from dataclasses import dataclass

import numpy as np

FP4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
FP8 = np.array([(n % 8) * 2.0 ** -9 if n < 8 else (8 + n % 8) * 2.0 ** (n // 8 - 10) for n in range(127)], np.float64)
_GRID = {"fp4": FP4, "fp8": FP8}
NAN_BITS = {"f16": 0x7E00, "bf16": 0x7FC0}
#: half a step of the 16-bit types, relative
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@np.errstate(invalid="ignore")  # signalling NaN patterns
def to_f64(x, dtype):
    x = np.asarray(x)
    if dtype == "f16":
        return x.view(np.float16).astype(np.float64)
    return (x.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def bits_of(x, dtype):
    """16-bit patterns of float64 values that the type holds, or of the nearest (ties to even)."""
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    f = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    r = ((f + 0x7FFF + ((f >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(NAN_BITS["bf16"]), r)


def quantise(x, fmt, dtype):
    """[..][D] in 16 bits -> (codes [..][blocks][32], one code an entry, scale bytes [..][blocks])."""
    v = to_f64(x, dtype)
    v = np.concatenate([v, np.zeros(v.shape[:-1] + (-v.shape[-1] % 32,))], -1)
    v = v.reshape(v.shape[:-1] + (v.shape[-1] // 32, 32))
    bad = ~np.isfinite(v).all(-1)
    most = (1.5 if fmt == "fp4" else 1.875) * 2.0 ** (15 if dtype == "f16" else 127)
    v = np.clip(np.where(bad[..., None], 0.0, v), -most, most)
    top, grid = np.abs(v).max(-1), _GRID[fmt]
    with np.errstate(divide="ignore"):
        e = np.maximum(np.where(top > 0, np.ceil(np.log2(np.where(top > 0, top, 1.0) / grid[-1])), -126.0), -126.0)
    e = np.where(top > grid[-1] * 2.0 ** e, e + 1, e)
    e = np.where((e > -126) & (top <= grid[-1] * 2.0 ** (e - 1)), e - 1, e)
    a = np.abs(v) * 2.0 ** -e[..., None]
    mid = (grid[1:] + grid[:-1]) / 2
    code = np.searchsorted(mid, a, "left")  # a tie falls on the lower code
    tie = (code < len(mid)) & (a == mid[np.minimum(code, len(mid) - 1)]) & (code % 2 == 1)
    code = code + tie + np.where(np.signbit(v), len(grid) + (0 if fmt == "fp4" else 1), 0)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def dequantise(codes, scales, fmt):
    """(codes [..][blocks][32], scale bytes) -> values [..][blocks * 32] in 64 bits."""
    g = _GRID[fmt]
    table = np.concatenate([g, -g]) if fmt == "fp4" else np.concatenate([g, [np.nan], -g, [np.nan]])
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    v = table[codes] * s[..., None]
    return v.reshape(v.shape[:-2] + (32 * v.shape[-2],))


@dataclass
class Cache:
    """A cache of n_pages pages on the host: `bytes`, laid out as the library's."""
    n_pages: int
    page: int
    H_kv: int
    D: int
    fmt: str
    dtype: str
    bytes: np.ndarray = None

    def __post_init__(self):
        self.blocks = -(-self.D // 32)
        self.row = self.blocks * (16 if self.fmt == "fp4" else 32)
        self.region = 2 * self.page * (self.row + self.blocks)
        if self.bytes is None:
            self.bytes = np.zeros(self.n_pages * self.H_kv * self.region, np.uint8)

    def part(self, which, scales):
        """View [page][head][position][byte] of the codes or scales of K (0) or V (1)."""
        width = self.blocks if scales else self.row
        at = self.page * ((2 * self.row + which * self.blocks) if scales else which * self.row)
        all_ = self.bytes.reshape(self.n_pages, self.H_kv, self.region)
        return all_[:, :, at:at + self.page * width].reshape(self.n_pages, self.H_kv, self.page, width)

    def put(self, which, page, off, x):
        """One position's rows [H_kv][D]."""
        codes, scales = quantise(x, self.fmt, self.dtype)
        flat = codes.reshape(self.H_kv, -1)
        if self.fmt == "fp4":
            flat = flat[:, 0::2] | (flat[:, 1::2] << 4)
        all_ = self.bytes.reshape(self.n_pages, self.H_kv, self.region)
        at = which * self.page * self.row + off * self.row
        all_[page, :, at:at + self.row] = flat
        at = self.page * (2 * self.row + which * self.blocks) + off * self.blocks
        all_[page, :, at:at + self.blocks] = scales

    def values(self, which, page, off):
        """Values of positions (page[n], off[n]), page -1 reading as NaN: [n][H_kv][D]."""
        ok = page >= 0
        p = np.where(ok, page, 0)
        codes = self.part(which, False)[p, :, off]
        if self.fmt == "fp4":
            codes = np.stack([codes & 15, codes >> 4], -1)
        v = dequantise(codes.reshape(codes.shape[0], self.H_kv, self.blocks, 32), self.part(which, True)[p, :, off], self.fmt)
        return np.where(ok[:, None, None], v[..., :self.D], np.nan)

    def pages_of(self, table_row, pos):
        """The page of each position, -1 where there is none."""
        pos = np.asarray(pos, np.int64)
        k = pos // self.page
        ok = (pos >= 0) & (k < len(table_row))
        page = np.where(ok, np.asarray(table_row)[np.clip(k, 0, len(table_row) - 1)], -1)
        return np.where((page >= 0) & (page < self.n_pages), page, -1)

    # ---- the three operators

    def _rows(self, T, row_start, kv_len):
        """(sequence, first row, rows, position of the first) with the library's limits on what the arrays hold."""
        for b in range(len(kv_len)):
            first = min(max(int(row_start[b]), 0), T)
            n = min(max(int(row_start[b + 1]), first), T) - first
            yield b, first, n, int(kv_len[b]) - n

    def write(self, K, V, row_start, kv_len, table):
        for b, first, n, pos0 in self._rows(len(K), row_start, kv_len):
            page = self.pages_of(table[b], pos0 + np.arange(n))
            for i in range(n):
                if page[i] >= 0:
                    self.put(0, page[i], (pos0 + i) % self.page, K[first + i])
                    self.put(1, page[i], (pos0 + i) % self.page, V[first + i])

    def read(self, T, row_start, kv_len, table, fill):
        """16-bit patterns of (K, V), `fill` in rows of no sequence."""
        out = [np.full((T, self.H_kv, self.D), fill, np.uint16) for _ in range(2)]
        for b, first, n, pos0 in self._rows(T, row_start, kv_len):
            pos = pos0 + np.arange(n)
            page = self.pages_of(table[b], pos)
            for w in range(2):
                out[w][first:first + n] = bits_of(self.values(w, page, pos % self.page), self.dtype)
        return out

    def attention(self, Q, row_start, kv_len, table, causal=True, S_q=0, only=None):
        """(O, lse, bound) in 64 bits; rows of no sequence are NaN with bound -1 (not computed), and so are rows that are not
        in `only`, if it is given. `bound` is what O may
        be off: half a step of the result; the weights' rounding, half a step of each; and the scores in 32 bits: D + 3
        roundings of 2^-24 of sum |q k| and of the scaled score and its offset, which move a weight by as much.
        f16 weights below 2^-14 have steps of 2^-24 whatever their value, so that half a step is 2^-25. Of some keys of a row the
        largest weight is held as 2^7 or more, so that this is at most 2^-25 / 2^7 = 2^-32 of the row's largest weight
        (of w below, whose largest is 1)."""
        T, H, D = Q.shape
        G, u = H // self.H_kv, HALF_STEP[self.dtype]
        q = to_f64(Q, self.dtype)
        O, lse, bound = np.full(Q.shape, np.nan), np.full((T, H), np.nan), np.full(Q.shape, -1.0)
        for b, first, n, pos0 in self._rows(T, row_start, kv_len):
            cap = len(table[b]) * self.page
            keys = min(max(int(kv_len[b]), 0), cap)
            pos = np.arange(keys)
            page = self.pages_of(table[b], pos)
            if kv_len[b] > cap:
                page[:] = -1
            k, v = (self.values(w, page, pos % self.page) for w in range(2))
            for i in range(min(n, S_q or T)):
                if only is not None and first + i not in only:
                    continue
                m = max(0, min(keys, pos0 + i + 1)) if causal else keys
                for h in range(H):
                    x = q[first + i, h]
                    if m == 0:
                        O[first + i, h], lse[first + i, h], bound[first + i, h] = 0.0, -np.inf, 0.0
                        continue
                    kk, vv = k[:m, h // G], v[:m, h // G]
                    s = kk @ x / np.sqrt(D)
                    top = s.max()
                    w = np.exp(s - top)
                    total = w.sum()
                    o = (w @ vv) / total
                    spread = np.abs(w) @ np.abs(vv) / total
                    slip = 2.0 ** -24 * ((D + 3) * (np.abs(kk) @ np.abs(x)).max() / np.sqrt(D) + 4 * np.abs(s).max() + 8)
                    O[first + i, h] = o
                    lse[first + i, h] = top + np.log(total) if top > -np.inf else top
                    # 32-bit sums over m keys: pairwise in the matrix unit and over tiles, at most m / 32 + 8 steps
                    sums = 2.0 ** -24 * (m / 32 + 8)
                    small = 2.0 ** -32 * np.abs(vv).sum(0) / total if self.dtype == "f16" else 0.0
                    bound[first + i, h] = u * np.abs(o) + ((u + 2 * slip + 2 * sums) * spread + small) * (1 + u) + 2.0 ** -24
        return O, lse, bound
