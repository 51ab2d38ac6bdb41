"""Attention over the 8-bit cache element by element: 64-bit results with the
sizes that an fp32 computation's errors are measured by, and the bound."""
import numpy as np
import torch

from tests.q8_util import BLOCK

# significand bits, the leading one among them
BITS = {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}
LEAST = {torch.float32: -125, torch.bfloat16: -125, torch.float16: -13}  # frexp's exponent of the least normal number


class Exact:
    """Attention of q [rows, heads, hd] over k, v [kvh, len, hd] in 64 bits;
    row j sees positions < seen[j] that are not hidden.
    out: the result; size: sum p |v|; most: scale * sum |q k| of the row's
    largest visible score; floor: sum over t of |v_t| times the largest weight
    in t's block of 16; floor_tiles: sum over t of |v_t| / step_t times the
    row's largest p * step (step [kvh, len]: what a position's value codes
    count in)."""

    def __init__(self, q, k, v, seen, hidden, scale, step):
        rows, heads, hd = q.shape
        kvh, n = k.shape[:2]
        g = heads // kvh
        shape = (rows, heads, hd)
        self.out, self.size, self.floor, self.floor_tiles = (np.zeros(shape) for _ in range(4))
        self.most = np.zeros((rows, heads, 1))
        show = np.arange(n)[None, :] < np.asarray(seen)[:, None]
        if hidden is not None:
            show = show & ~np.asarray(hidden, bool)[None, :n]
        pad = -n % BLOCK
        for h in range(heads):
            kk, vv = k[h // g], v[h // g]
            with np.errstate(all="ignore"):
                s = scale * (q[:, h] @ kk.T)
                a = abs(scale) * (np.abs(q[:, h]) @ np.abs(kk).T)
            s = np.where(show, s, -np.inf)
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.where(show, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(1, keepdims=True)
            p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
            seen_v = np.where(show.any(0)[:, None], vv, 0.0)  # what no row sees may be no number
            blk = np.pad(p, ((0, 0), (0, pad))).reshape(rows, -1, BLOCK).max(2).repeat(BLOCK, 1)[:, :n]
            self.out[:, h] = p @ seen_v
            self.size[:, h] = p @ np.abs(seen_v)
            self.floor[:, h] = np.where(show, blk, 0.0) @ np.abs(seen_v)
            z = np.maximum(step[h // g], 2.0 ** -130)
            part = np.where(show, p * z, 0.0).max(1, keepdims=True, initial=0.0)
            self.floor_tiles[:, h] = np.where(show, part / z, 0.0) @ np.abs(seen_v)
            self.most[:, h, 0] = np.where(show, a, 0.0).max(1, initial=0.0)

    def bound(self, dtype, got, tiles=False):
        """How far an element may be off. Scores: a sum whose terms add up to
        at most `most`, 8 roundings of 2^-24 of it counted; the exponential,
        the weight's rounding to two 11-bit terms (2^-22), the sums of at most
        40 partial results and the quotient: 64 roundings of 2^-24. Both count
        in the numerator and in the denominator. A weight's second term ends at
        2^-24 where the largest weight of its block is 2^14 or more (the tiles:
        where the row's largest weight times step is 2^10 or more): half of
        that. And the result's rounding."""
        d = 2 * (8 * self.most + 64) * 2.0 ** -24 * self.size
        d += 2.0 ** -35 * self.floor_tiles if tiles else 2.0 ** -39 * self.floor
        big = np.maximum(np.abs(got), np.abs(self.out))
        _, e = np.frexp(big)
        return d + np.where(big > 0, np.exp2(np.maximum(e, LEAST[dtype]).astype(float) - 1 - BITS[dtype]), 0.0)

    def worst(self, got, dtype, tiles=False):
        """Largest difference over its bound (1 or less is right)."""
        got = got.double().cpu().numpy()
        off = np.abs(got - self.out)
        b = self.bound(dtype, got, tiles)
        with np.errstate(all="ignore"):
            r = np.where(off == 0, 0.0, off / b)
        return np.nan_to_num(r, nan=np.inf).max(initial=0.0)
