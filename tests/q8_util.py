"""A plain 8-bit key/value cache for the tests: the tokens as given, their
codes by the definition in numpy fp32 steps, attention in 64 bits."""
import numpy as np
import torch

BLOCK = 16
TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def quantise(x, kind):
    """(codes as float values, scale) of one block x [16, hd] (float32 numpy)."""
    top = np.float32(TOP[kind])
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        fine = np.isfinite(x)
        a = np.abs(np.where(fine, x, np.float32(0))).max().astype(np.float32)
        s = np.float32(0) if a < np.float32(2.0 ** -117) else np.float32(a / top)
        r = np.float32(1) / s if s > 0 else np.float32(0)
        t = (x * r).astype(np.float32)
        t = np.clip(np.where(np.isnan(t), np.float32(0), t), -top, top)
    if kind == "int8":
        return np.rint(t), s
    # e4m3: 3 mantissa bits above 2^-6, steps of 2^-9 below
    e = np.floor(np.log2(np.maximum(np.abs(t).astype(np.float64), 2.0 ** -6)))
    step = 2.0 ** (e - 3)
    return np.clip(np.rint(t.astype(np.float64) / step) * step, -448, 448).astype(np.float32), s


class Plain:
    """One sequence's K or V: the rows as given, [len, kv_heads, hd] fp32."""

    def __init__(self, kvh, hd, kind, dtype):
        self.kind, self.dtype = kind, dtype
        self.x = np.zeros((0, kvh, hd), np.float32)

    def append(self, rows):
        self.x = np.concatenate([self.x, rows.float().cpu().numpy()])

    def closed(self):
        """(codes as values [kvh, nb, 16, hd], scales [kvh, nb])."""
        n, kvh, hd = self.x.shape
        nb = n // BLOCK
        c = np.zeros((kvh, nb, BLOCK, hd), np.float32)
        s = np.zeros((kvh, nb), np.float32)
        for h in range(kvh):
            for b in range(nb):
                c[h, b], s[h, b] = quantise(self.x[b * BLOCK:(b + 1) * BLOCK, h], self.kind)
        return c, s

    def values(self):
        """fp64 [kvh, len, hd]: what the cache holds."""
        n, kvh, hd = self.x.shape
        c, s = self.closed()
        v = (c.astype(np.float64) * s[..., None, None]).reshape(kvh, -1, hd)
        return np.concatenate([v, self.x[n // BLOCK * BLOCK:].transpose(1, 0, 2).astype(np.float64)], 1)


def attend64(q, k, v, seen, hidden, scale):
    """fp64 attention of q [rows, heads, hd] over k, v [kvh, len, hd]: row j
    sees positions < seen[j] that are not hidden. Returns (out, A) with A the
    largest scale * sum |q k| of a visible score."""
    rows, heads, hd = q.shape
    kvh, n = k.shape[:2]
    g = heads // kvh
    out = np.zeros((rows, heads, hd))
    most = 0.0
    show = np.arange(n)[None, :] < np.asarray(seen)[:, None]
    if hidden is not None:
        show &= ~hidden[None, :n].astype(bool)
    for h in range(heads):
        kk, vv = k[h // g], v[h // g]
        for j in range(rows):
            at = show[j]
            if not at.any():
                continue
            s = scale * (kk[at] @ q[j, h])
            most = max(most, float((abs(scale) * np.abs(kk[at]) @ np.abs(q[j, h])).max()))
            p = np.exp(s - s.max())
            out[j, h] = (p / p.sum()) @ vv[at]
    return out, most


def tolerance(dtype, most):
    """2-norm bound of the attention's relative error. fp32 steps: a score is
    a sum whose terms add up to at most `most`, each product and addition off
    by 2^-24 of it (8 of them counted: they are of either sign), so a weight
    is off by 8 * most * 2^-24, plus 16 roundings of the exponential, the
    sums and the quotient. 16-bit results add half a step for the output and
    2^-12 for weights rounded to 11 bits."""
    t = (8 * most + 16) * 2.0 ** -24
    if dtype != torch.float32:
        t += torch.finfo(dtype).eps / 2 + 2.0 ** -12
    return t


def far(got, want):
    """2-norm of the difference over the 2-norm of what is wanted."""
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    norm = np.linalg.norm(want)
    off = np.linalg.norm(got - want)
    return off / norm if norm else (0.0 if off == 0 else np.inf)
