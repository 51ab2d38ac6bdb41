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


def steps(c, slot, hidden=None):
    """What the value codes of a slot's positions count in, [kvh, len]: the
    block's scale; in the open block 2^-6 of its largest visible value, or as
    little as 2^-15 of it where its smallest ones need that to keep their bits
    above 2^-24."""
    p = c.plain[slot][1]
    s = p.closed()[1].astype(float).repeat(BLOCK, 1)
    x = np.abs(p.x[s.shape[1]:].astype(float))  # [open positions, kvh, hd]
    if hidden is not None:
        x = np.where(np.asarray(hidden, bool)[s.shape[1]:len(p.x), None, None], 0.0, x)
    x = np.where(np.isfinite(x), x, 0.0)
    top = x.max((0, 2), initial=0.0)
    low = np.where(x > 0, x, np.inf).min((0, 2), initial=np.inf)
    with np.errstate(all="ignore"):
        e, f = np.floor(np.log2(top)), np.floor(np.log2(low))
        last = np.maximum(f - 10, -24) if c.dtype == F16 else f - 7
        z = np.where(top > 0, np.exp2(e - np.clip(e - last - 24, 6, 15)), 1.0)
    return np.concatenate([s, np.repeat(z[:, None], len(x), 1)], 1)


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
                  None if hidden is None else hidden[i], sc, steps(c, s, None if hidden is None else hidden[i]))
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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("hd", [64, 128])
def test_values_near_the_largest_number(dtype, kind, rows, hd):
    c = Case(5, 1, 192, hd, kind, dtype, seed=9)
    lens = [1, 10, 160, 171, 175]
    # the tiles hold a block's values as 16-bit numbers in units of its largest: no dims 2^40 below it
    tiles = on_tiles(dtype, hd, rows, 4)
    v = c.randn(sum(lens), 1, hd)
    v[0] = v[0] * 1e37 if tiles else v[0]
    v[0, 0, 7] = 2e38                                            # alone
    v[1:11] = (v[1:11].float().clamp(-3, 3) * 1e38).to(dtype)    # the open block alone
    v[11:171] = (v[11:171].float().clamp(-3, 3) * 1e38).to(dtype)  # closed blocks alone
    at = 171
    v[at + 165, 0, 3] = 3e38                                     # one in the open block, ordinary ones before it
    at += 171
    v[at:at + 175] = (v[at:at + 175].float().clamp(-3, 3) * 1e38).to(dtype)
    c.append([0, 1, 2, 3, 4], lens, c.randn(sum(lens), 1, hd), v)
    out = check(c, [0, 1, 2, 4] if tiles else [0, 1, 2, 3, 4], rows, 4, causal=False)
    assert torch.isfinite(out).all()
    check(c, [4, 2], rows, 4)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("where", [50, 171])
def test_one_value_that_dwarfs_the_others_leaves_their_dims_alone(dtype, rows, hd, where):
    """`where`: a closed block, the open one. 1e9 times the others (the tiles: 2^14 times)."""
    c = Case(1, 2, 192, hd, "int8", dtype, seed=10)
    k, v = c.randn(174, 2, hd), c.randn(174, 2, hd)
    v[where, :, 5] = 2.0 ** 14 if on_tiles(dtype, hd, rows, 2) else 1e9
    c.append([0], [174], k, v)
    check(c, [0], rows, 4, causal=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 140])
def test_small_elements_of_the_open_block(dtype, rows):
    """Elements 2^16 to 2^24 below the largest of the open block keep their bits."""
    for hd in (64, 128):
        c = Case(1, 1, 32, hd, "int8", dtype, seed=11)
        v = c.randn(13, 1, hd).float()
        v = v.clamp(-3, 3) * torch.exp2(-(torch.arange(hd, device="cuda") % 9).float())
        v = v * 2.0 ** -3
        v[4, 0, 0] = 2.0 ** 13
        k = c.randn(13, 1, hd)
        c.append([0], [13], k, v.to(dtype))
        check(c, [0], rows, 2, causal=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("at", [20, 166])
def test_keys_near_the_largest_number(dtype, rows, at):
    """Scores far beyond what an exponential can hold: the largest one's value, whatever the values' size."""
    for size in (1.0, 1e6, 1e30):
        c = Case(1, 1, 192, 64, "int8", dtype, seed=12)
        k, v = c.randn(170, 1, 64), (c.randn(170, 1, 64).float() * size).to(dtype)
        k[at, 0, 2] = 1e35
        c.append([0], [170], k, v)
        q = c.randn(rows, 2, 64)
        q[..., 2] = 1.0
        out = torch.empty_like(q)
        D.q8_attend(c.cache, q, out, ints([170]), causal=False)
        want = torch.tensor(c.values(0)[1][0, at], device="cuda").to(dtype)
        step = torch.finfo(dtype).eps
        bad = ((out - want).abs() > step * want.abs()) | torch.isnan(out)
        assert bad.sum().item() == 0, (size, out[0, 0, :4].tolist(), want[:4].tolist())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_an_ordinary_open_block_beside_large_values(dtype, hd):
    """Tiles: a closed block's value 2^13 times the others leaves the open block's weights their bits."""
    c = Case(1, 1, 64, hd, "int8", dtype, seed=13)
    k, v = c.randn(47, 1, hd), c.randn(47, 1, hd)
    v[:32] = 0
    v[5, 0, 3] = 2.0 ** 13
    c.append([0], [47], k, v)
    check(c, [0], 140, 4, causal=False)
