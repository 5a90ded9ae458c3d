"""Products grouped by expert, and rows and products in few bits (include/mtk.h), in numpy and 64 bits: the plain
implementations that the tests compare with. f16 tensors are numpy float16 patterns, bf16 tensors uint16 bit patterns."""
import numpy as np

from . import kv

HALF_STEP = kv.HALF_STEP
#: half the distance of the smallest subnormals
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def spans(row_start, T):
    """[(first, end)] of each group, whatever row_start holds."""
    out = []
    for i, j in zip(row_start[:-1], row_start[1:]):
        first = min(max(int(i), 0), T)
        out.append((first, min(max(int(j), first), T)))
    return out


def _bound(y, mag, terms, kind):
    """What a result in `kind` may be off by: half a step of it, and of its fp32 sum of `terms` products (exact in fp32, being
    of 16 or fewer bits), whose magnitudes add up to mag. Every addition is off by at most one unit in the last place of a
    partial sum, 2^-23 of at most mag, however the hardware orders and rounds them; the bias is one more."""
    off = (terms + 1) * 2.0 ** -23 * mag + 2.0 ** -149 * terms
    if kind == "f32":
        return off
    return off + HALF_STEP[kind] * (np.abs(y) + off) + TINY[kind]


def grouped(A, B, bias, row_start, trans_b, dtype):
    """(C [T][N], bound, rows that a group has) in 64 bits."""
    a, b = kv.to_f64(A, dtype), kv.to_f64(B, dtype)
    T, K = a.shape
    N = b.shape[1] if trans_b else b.shape[2]
    y, mag, mine = np.zeros((T, N)), np.zeros((T, N)), np.zeros(T, bool)
    for e, (i, j) in enumerate(spans(row_start, T)):
        w = b[e].T if trans_b else b[e]
        y[i:j], mag[i:j], mine[i:j] = a[i:j] @ w, np.abs(a[i:j]) @ np.abs(w), True
        if bias is not None:
            v = kv.to_f64(bias[e], dtype)
            y[i:j] += v
            mag[i:j] += np.abs(v)
    return y, _bound(y, mag, K, dtype), mine


def grad(A, dC, row_start, trans_b, dtype, out):
    """((dB, bound), (dbias, bound)) in 64 bits; out: "f32" or the type."""
    a, d = kv.to_f64(A, dtype), kv.to_f64(dC, dtype)
    T, K = a.shape
    N = d.shape[1]
    parts = []
    for i, j in spans(row_start, T):
        x, g = a[i:j], d[i:j]
        l, r = (g, x) if trans_b else (x, g)
        y, b = l.T @ r, g.sum(0)
        parts.append((y, _bound(y, np.abs(l).T @ np.abs(r), j - i, out), b, _bound(b, np.abs(g).sum(0), j - i, out)))
    pick = lambda n: np.stack([p[n] for p in parts])
    return (pick(0), pick(1)), (pick(2), pick(3))


def quantise(x, dtype):
    """Rows [R][K] in 16 bits -> (codes [R][k_tiles * 128], scales [k_tiles][R][8]), bytes as the library lays them out."""
    x = np.asarray(x)
    R, K = x.shape
    x = np.concatenate([x.view(np.uint16), np.zeros((R, -K % 256), np.uint16)], 1)
    codes, scales = kv.quantise(x, "fp4", dtype)
    codes = codes.reshape(R, -1)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), np.ascontiguousarray(scales.reshape(R, -1, 8).transpose(1, 0, 2))


def values(codes, scales, K):
    """The values [R][K] that codes and scales stand for, in 64 bits."""
    R = codes.shape[0]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(R, -1, 32)
    return kv.dequantise(c, scales.transpose(1, 0, 2).reshape(R, -1), "fp4")[:, :K]


def mx_product(a, b, bias, row_start, dtype):
    """Values a [T][K], b [E][N][K] in 64 bits -> (C, bound, rows that a group has). The products of e2m1 values are exact."""
    T, K = a.shape
    N = b.shape[1]
    y, mag, mine = np.zeros((T, N)), np.zeros((T, N)), np.zeros(T, bool)
    for e, (i, j) in enumerate(spans(row_start, T)):
        y[i:j], mag[i:j], mine[i:j] = a[i:j] @ b[e].T, np.abs(a[i:j]) @ np.abs(b[e]).T, True
        if bias is not None:
            v = kv.to_f64(bias[e], dtype)
            y[i:j] += v
            mag[i:j] += np.abs(v)
    return y, _bound(y, mag, K, dtype), mine
