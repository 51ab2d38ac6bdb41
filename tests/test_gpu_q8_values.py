"""Attention over the 8-bit cache, element by element against 64 bits: what a
2-norm over a whole result cannot see."""
import numpy as np
import pytest

import defer_b200 as D
from tests.q8_exact import Exact
from tests.q8_util import BLOCK
from tests.test_gpu_q8 import Case, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def on_tiles(dtype, hd, rows, group):
    return dtype != F32 and hd <= 128 and rows * group > 64


def steps(c, slot):
    """What the value codes of a slot's positions count in, [kvh, len]: the
    block's scale; in the open block 2^-15 of its largest value."""
    p = c.plain[slot][1]
    s = p.closed()[1].astype(float).repeat(BLOCK, 1)
    x = np.abs(p.x[s.shape[1]:].astype(float))  # [open positions, kvh, hd]
    a = x.max((0, 2), initial=0.0, where=np.isfinite(x))
    return np.concatenate([s, np.repeat(a[:, None] * 2.0 ** -15, len(x), 1)], 1)


def check(c, slots, rows, heads, q=None, hidden=None, scale=None, causal=True, **kw):
    """Attention of `rows` random rows of each slot; returns the output."""
    q = c.randn(len(slots) * rows, heads, c.hd) if q is None else q
    out = torch.full_like(q, 77.0)
    lens = [c.len(s) for s in slots]
    masked = None
    if hidden is not None:
        masked = torch.zeros(len(slots), c.cap, dtype=torch.uint8, device="cuda")
        for i, h in enumerate(hidden):
            masked[i, :len(h)] = torch.tensor(h, dtype=torch.uint8, device="cuda")
    D.q8_attend(c.cache, q, out, ints(lens), slots=ints(slots), masked=masked, scale=scale, causal=causal,
                **kw)
    sc = c.hd ** -0.5 if scale is None else scale
    for i, s in enumerate(slots):
        k, v = c.values(s)
        seen = [lens[i] - (rows - 1 - j) if causal else lens[i] for j in range(rows)]
        e = Exact(q[i * rows:(i + 1) * rows].double().cpu().numpy(), k, v, seen,
                  None if hidden is None else hidden[i], sc, steps(c, s))
        w = e.worst(out[i * rows:(i + 1) * rows], c.dtype, on_tiles(c.dtype, c.hd, rows, heads // c.kvh))
        assert w <= 1, (i, s, lens[i], w)
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 5, 140])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (4, 2, 128), (2, 1, 32)])
def test_weights_keep_more_bits_than_the_result(dtype, kind, rows, heads, kvh, hd):
    """Every element is the exact one rounded once, up to the errors of an fp32 computation."""
    c = Case(4, kvh, 352, hd, kind, dtype, seed=hd + rows)
    c.append([0, 1, 2, 3], [150, 40, 345, 208])
    check(c, [2, 0, 3, 1], rows, heads)
