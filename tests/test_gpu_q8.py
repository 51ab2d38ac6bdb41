"""8-bit key/value cache on the GPU against the plain one of q8_util: codes,
scales and values bit for bit, attention in 64 bits at the derived tolerance,
at the sizes, masks and layouts where it can go wrong."""
import numpy as np
import pytest

import defer_b200 as D
from tests.q8_util import BLOCK, CODE, Plain, attend64, far, tolerance

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    """A cache on the GPU and its plain twin, slot by slot."""

    def __init__(self, slots, kvh, cap, hd, kind, dtype, seed=0):
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.kvh, self.hd, self.kind, self.dtype, self.cap = kvh, hd, kind, dtype, cap
        # what no call has written holds NaN codes' bytes, NaN scales and NaN tails: none of it may be used
        self.codes = [torch.full((slots, kvh, cap, hd), 0x7F, dtype=torch.int8, device="cuda").view(CODE[kind])
                      for _ in range(2)]
        self.scales = [torch.full((slots, kvh, cap // BLOCK), float("nan"), device="cuda") for _ in range(2)]
        self.tails = [torch.full((slots, kvh, BLOCK, hd), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
        self.cache = D.Q8Cache(*self.codes, *self.scales, *self.tails)
        self.plain = [[Plain(kvh, hd, kind, dtype) for _ in range(2)] for _ in range(slots)]

    def randn(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.g).to(self.dtype)

    def len(self, slot):
        return len(self.plain[slot][0].x)

    def append(self, slots, counts, k=None, v=None, **kw):
        k = self.randn(sum(counts), self.kvh, self.hd) if k is None else k
        v = self.randn(sum(counts), self.kvh, self.hd) if v is None else v
        at = np.concatenate([[0], np.cumsum(counts)]).tolist()
        D.q8_append(self.cache, k, v, ints([self.len(s) if s >= 0 else 0 for s in slots]), q_start=ints(at),
                    slots=ints(slots), max_q=max(counts), **kw)
        for i, s in enumerate(slots):
            if s >= 0:
                self.plain[s][0].append(k[at[i]:at[i + 1]])
                self.plain[s][1].append(v[at[i]:at[i + 1]])

    def check(self):
        """Codes, scales and tails of every slot, bit for bit."""
        for s, pair in enumerate(self.plain):
            for x, p in enumerate(pair):
                n = len(p.x)
                nb = n // BLOCK
                c, z = p.closed()
                got = self.codes[x][s].float().cpu().numpy().reshape(self.kvh, -1, BLOCK, self.hd)
                assert np.array_equal(got[:, :nb], c), (s, x)
                assert np.array_equal(self.scales[x][s].cpu().numpy()[:, :nb], z), (s, x)
                assert torch.isnan(self.scales[x][s][:, nb:]).all()
                assert (self.codes[x][s].view(torch.int8)[:, nb * BLOCK:] == 0x7F).all()
                tail = self.tails[x][s].float().cpu().numpy()[:, :n - nb * BLOCK]
                assert np.array_equal(tail, p.x[nb * BLOCK:].transpose(1, 0, 2), equal_nan=True), (s, x)

    def values(self, slot):
        return [p.values() for p in self.plain[slot]]

    def attend_check(self, slots, counts, heads, causal=True, hidden=None, scale=None, q=None, **kw):
        """Attention of random rows against 64 bits; returns the output."""
        tokens = sum(counts)
        q = self.randn(tokens, heads, self.hd) if q is None else q
        out = torch.full_like(q, 77.0)
        at = np.concatenate([[0], np.cumsum(counts)]).tolist()
        lens = [self.len(s) if s >= 0 else 0 for s in slots]
        masked = None
        if hidden is not None:
            masked = torch.zeros(len(slots), self.cap, dtype=torch.uint8, device="cuda")
            for i, h in enumerate(hidden):
                masked[i, :len(h)] = torch.tensor(h, dtype=torch.uint8, device="cuda")
        D.q8_attend(self.cache, q, out, ints(lens), q_start=ints(at), slots=ints(slots), masked=masked, causal=causal,
                    scale=scale, **kw)
        sc = self.hd ** -0.5 if scale is None else scale
        for i, s in enumerate(slots):
            got = out[at[i]:at[i + 1]]
            if s < 0:
                assert (got == 77.0).all()
                continue
            k, v = self.values(s)
            seen = [lens[i] - (counts[i] - 1 - j) if causal else lens[i] for j in range(counts[i])]
            h = None if hidden is None else np.pad(np.asarray(hidden[i], bool), (0, max(0, lens[i] - len(hidden[i]))))
            want, most = attend64(q[at[i]:at[i + 1]].double().cpu().numpy(), k, v, seen, h, sc)
            e = far(got, want)
            assert e <= tolerance(self.dtype, most), (i, s, lens[i], counts[i], e, tolerance(self.dtype, most))
        return out


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 256])
def test_append_writes_the_definitions_codes(dtype, kind, hd):
    c = Case(4, 2, 96, hd, kind, dtype, seed=hd)
    c.append([2, 0, 1], [1, 17, 40])       # inside a block, across one border, across two
    c.check()
    c.append([0, 1, 2, 3], [15, 0, 31, 16])  # closes with the tail's tokens; none; ends on a border; a whole block
    c.check()
    c.append([3, -1, 2], [33, 5, 1])       # sequence 1 is padding
    c.check()


def test_append_in_pieces_gives_the_same_bits():
    k = [torch.randn(70, 3, 64, device="cuda") * 3 for _ in range(2)]
    whole, steps = Case(1, 3, 80, 64, "int8", F32), Case(1, 3, 80, 64, "int8", F32)
    whole.append([0], [70], *k)
    done = 0
    for n in [1] * 18 + [5, 2, 30, 15]:
        steps.append([0], [n], *(x[done:done + n] for x in k))
        done += n
    assert done == 70
    for a, b in zip(whole.codes, steps.codes):
        assert torch.equal(a, b)
    for a, b in zip(whole.scales, steps.scales):
        assert torch.equal(a[..., :4], b[..., :4])
    steps.check()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_of_special_values(kind):
    c = Case(1, 1, 160, 64, kind, F32)
    x = torch.randn(144, 1, 64, device="cuda")
    x[3, 0, 5], x[3, 0, 6] = float("nan"), float("inf")
    x[4, 0, 7] = -float("inf")
    x[16:32] = 0                               # zeros
    x[32:48] *= 1e-40                          # below the smallest scale
    x[48:64] = 3.0e38 * torch.sign(x[48:64])   # near the largest number
    x[64:80] = float("nan")                    # nothing finite
    x[80:96] *= 2.0 ** -110                    # a small scale that is kept
    x[96:112] = torch.round(x[96:112] * 4) / 4 # values on rounding borders
    x[112:128, :, 0] = 1e6                     # one channel dwarfs the others
    c.append([0], [144], x, torch.flip(x, [2]).contiguous())
    for p in c.plain[0]:
        assert np.isfinite(p.values()[:, :144]).all()
    c.check()


def test_append_from_strided_and_unaligned_rows():
    c = Case(2, 3, 64, 64, "int8", BF16)
    buf = c.randn(40, 2, 3, 65)  # rows of 65: no 16-byte alignment; k and v interleaved
    c.append([1, 0], [22, 18], buf[:, 0, :, 1:], buf[:, 1, :, :64])
    c.check()
    c.append([1, 0], [10, 10], c.randn(3, 20, 64).transpose(0, 1), c.randn(20, 1, 64).expand(20, 3, 64))
    c.check()


def test_append_skips_what_is_out_of_range():
    c = Case(3, 2, 32, 64, "int8", F32)
    c.append([0, 1, 2], [5, 5, 5])
    status = ints([0])
    k = c.randn(12, 2, 64)
    q = ints([0, 3, 6, 9, 12])
    D.q8_append(c.cache, k, k, ints([5, -1, 30, 5]), q_start=q, slots=ints([3, 1, 2, 7]), status=status)
    assert status.item() == 1
    c.check()
    D.q8_append(c.cache, k, k, ints([5, 5]), q_start=ints([0, -1, 4]), slots=ints([0, 1]), status=status)
    D.q8_append(c.cache, k, k, ints([5]), q_start=ints([0, 13]), slots=ints([0]), status=status)
    D.q8_append(c.cache, k, k, ints([5]), q_start=ints([4, 2]), slots=ints([0]), status=status)
    c.check()
    # a slot named twice is written by the first
    status.zero_()
    D.q8_append(c.cache, k, k, ints([5, 5]), q_start=ints([0, 4, 12]), slots=ints([1, 1]), status=status)
    for p in c.plain[1]:
        p.append(k[:4])
    assert status.item() == 2
    c.check()


def test_append_without_q_start_and_with_a_small_max_q():
    c = Case(3, 2, 160, 64, "int8", F32)
    k = c.randn(150, 2, 64)
    D.q8_append(c.cache, k, k, ints([0, 0, 0]))
    for s in range(3):
        for p in c.plain[s]:
            p.append(k[50 * s:50 * s + 50])
    c.check()
    D.q8_append(c.cache, k[:100], k[:100], ints([50]), q_start=ints([0, 100]), slots=ints([1]), max_q=1)
    for p in c.plain[1]:
        p.append(k[:100])
    c.check()


# --------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 256])
def test_read_gives_the_values(dtype, kind, hd):
    c = Case(3, 2, 96, hd, kind, dtype, seed=hd)
    c.append([0, 1, 2], [16, 37, 90])
    for order in (0, 1):
        shape = (4, 95, 2, hd) if order else (4, 2, 95, hd)
        k, v = (torch.full(shape, 7.0, dtype=dtype, device="cuda") for _ in range(2))
        ko, vo = (k.transpose(1, 2), v.transpose(1, 2)) if order else (k, v)
        D.q8_read(c.cache, ko, vo, ints([37, 90, 0, 16]), slots=ints([1, 2, 0, -1]))
        for i, (s, n) in enumerate(((1, 37), (2, 90), (0, 0), (0, 0))):
            for got, want in zip((ko, vo), c.values(s)):
                w = torch.tensor(want[:, :n].astype(np.float32), device="cuda").to(dtype)
                assert torch.equal(got[i, :, :n], w)
                assert (got[i, :, n:] == 7.0).all()
    # a window, into rows that are not aligned
    k, v = (torch.full((2, 2, 20, hd + 1), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    D.q8_read(c.cache, k[..., 1:], v[..., 1:], ints([90, 37]), start=ints([75, 3]), slots=ints([2, 1]))
    for i, (s, a, n) in enumerate(((2, 75, 15), (1, 3, 20))):
        for got, want in zip((k, v), c.values(s)):
            w = torch.tensor(want[:, a:a + n].astype(np.float32), device="cuda").to(dtype)
            assert torch.equal(got[i, :, :n, 1:], w)
            assert (got[i, :, n:] == 7.0).all() and (got[..., 0] == 7.0).all()


def test_read_skips_what_is_out_of_range():
    c = Case(2, 1, 32, 64, "int8", F32)
    c.append([0, 1], [20, 20])
    k, v = (torch.full((4, 1, 32, 64), 7.0, device="cuda") for _ in range(2))
    status = ints([0])
    D.q8_read(c.cache, k, v, ints([33, -1, 20, 20]), start=ints([0, 0, -1, 0]), slots=ints([0, 1, 0, 2]), status=status)
    assert status.item() == 1 and (k == 7.0).all() and (v == 7.0).all()


# ------------------------------------------------------------------- attend
LENS = [1, 15, 16, 17, 31, 64, 127, 128, 129, 255, 300, 641]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kvh,hd", [(9, 3, 64), (4, 1, 128), (2, 2, 16), (8, 1, 256), (20, 2, 80), (32, 32, 32),
                                          (6, 2, 144), (4, 4, 48)])
def test_attend_single_rows(dtype, kind, heads, kvh, hd):
    c = Case(len(LENS), kvh, 656, hd, kind, dtype, seed=heads + hd)
    slots = list(range(len(LENS)))
    c.append(slots[::-1], LENS)
    c.attend_check(slots, [1] * len(slots), heads)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kvh,hd", [(9, 3, 64), (8, 2, 128), (3, 3, 64), (4, 2, 16), (8, 1, 256), (10, 2, 80)])
def test_attend_many_rows(dtype, kind, heads, kvh, hd):
    c = Case(6, kvh, 400, hd, kind, dtype, seed=hd)
    c.append(list(range(6)), [1, 40, 129, 200, 257, 397])
    # one row, none, more rows than fit a tile, all rows of a sequence, more rows than positions
    c.attend_check([3, 0, 5, -1, 2, 1, 4], [1, 0, 75, 3, 129, 44, 130], heads)
    c.attend_check([5, 1], [33, 2], heads, causal=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 5, 140])
def test_attend_hidden_positions(dtype, rows):
    c = Case(5, 2, 352, 64, "int8", dtype, seed=rows)
    c.append(list(range(5)), [345] * 5)
    r = np.random.default_rng(0)
    hidden = [r.random(345) < 0.3,                  # some
              np.ones(345, bool),                   # all: rows of zeros
              np.arange(345) < 330,                 # all closed blocks but the last
              np.arange(345) != 344,                # all but the newest
              np.arange(345) >= 7]                  # all but the oldest
    out = c.attend_check(list(range(5)), [rows] * 5, 6, hidden=hidden)
    assert (out[rows:2 * rows] == 0).all()
    # bool masks, and one mask for all sequences
    m = torch.tensor(np.pad(hidden[0], (0, 7)), device="cuda")
    q = c.randn(5 * rows, 6, 64)
    a, b = torch.empty_like(q), torch.empty_like(q)
    lens = ints([345] * 5)
    D.q8_attend(c.cache, q, a, lens, masked=m.expand(5, 352))
    D.q8_attend(c.cache, q, b, lens, masked=m.to(torch.uint8).repeat(5, 1))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 150])
def test_hidden_places_may_hold_anything(dtype, rows):
    """NaN, infinities and the type's lowest value in hidden and unwritten places change nothing."""
    heads, hd = 4, 64
    c = Case(2, 2, 192, hd, "e4m3", dtype, seed=3)
    k, v = c.randn(348, 2, hd), c.randn(348, 2, hd)
    low = torch.finfo(dtype).min
    for x in (k, v):
        x[5], x[40, :, 3], x[170], x[171] = float("nan"), float("inf"), float("nan"), low
        x[20:24] = low
    bad = np.zeros(174, bool)
    bad[[5, 40, 170, 171]] = True
    bad[16:48] = True  # their blocks' scales are the lowest values': hidden as a whole
    c.append([0, 1], [174, 174], torch.cat([k[:174], k[174:]]), torch.cat([v[:174], v[174:]]))
    out = c.attend_check([0, 1], [rows, rows], heads, hidden=[bad, np.zeros(174, bool)])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_and_tiny_scores_and_values(dtype):
    c = Case(4, 1, 192, 64, "int8", dtype, seed=8)
    k, v = c.randn(4 * 180, 1, 64), c.randn(4 * 180, 1, 64)
    k[180:360] *= 40                      # weights of one position alone
    v[180:360] *= 1e30
    v[360:540] *= 1e-25
    v[540:556] *= 1e6                     # one block's values dwarf the others', its keys are far away
    k[540:556] -= 100 * torch.sign(k[556:557])
    c.append([0, 1, 2, 3], [180] * 4, k, v)
    for rows in (1, 130):
        c.attend_check([0, 1, 2, 3], [rows] * 4, 2)
        c.attend_check([0, 1, 2, 3], [rows] * 4, 2, scale=-0.25)
        c.attend_check([0, 1, 2, 3], [rows] * 4, 2, scale=0.0)
        q = c.randn(4 * rows, 2, 64)
        q[:rows] *= 1e-30
        q[rows:2 * rows] = 0
        c.attend_check([0, 1, 2, 3], [rows] * 4, 2, q=q)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_a_non_finite_query_stays_in_its_row(dtype):
    for rows in (1, 140):
        c = Case(2, 1, 160, 64, "int8", dtype, seed=1)
        c.append([0, 1], [150, 150])
        q = c.randn(2 * rows, 4, 64)
        q[0, 1, 3], q[0, 3, 3] = float("nan"), float("inf")
        out = torch.empty_like(q)
        D.q8_attend(c.cache, q, out, ints([150, 150]))
        bad = torch.isnan(out).any(-1)
        assert bad[0, 1] and bad[0, 3] and bad.sum() == 2


def test_lengths_out_of_range_and_rows_behind():
    c = Case(3, 2, 32, 64, "int8", F32)
    c.append([0, 1, 2], [20, 20, 20])
    q = c.randn(9, 4, 64)
    for starts in ([0, 2, 4, 5, 7], [0, 2, 4, 5, 7]):
        out = torch.full_like(q, 77.0)
        status = ints([0])
        D.q8_attend(c.cache, q, out, ints([33, -1, 20, 20]), q_start=ints(starts), slots=ints([0, 1, 2, 3]),
                    status=status)
        assert status.item() == 1
        assert torch.isnan(out[:4]).all() and torch.isfinite(out[4]).all() and torch.isnan(out[5:7]).all()
        assert (out[7:] == 77.0).all()
    out = torch.full_like(q, 77.0)
    D.q8_attend(c.cache, q, out, ints([20, 20]), q_start=ints([0, 4, 10]), slots=ints([0, 1]))  # past the rows
    assert torch.isfinite(out[:4]).all() and (out[4:] == 77.0).all()
    D.q8_attend(c.cache, q, out, ints([0, 0, 0]))  # empty sequences
    assert (out == 0).all()


def test_visible_values_that_are_no_numbers():
    """A NaN or an infinity among the open block's values reaches the rows that see it, and only its own dim."""
    for dtype in (F32, BF16):
        for rows in (4, 140):
            c = Case(1, 1, 192, 64, "int8", dtype, seed=2)
            k, v = c.randn(172, 1, 64), c.randn(172, 1, 64)
            v[169, 0, 7], v[170, 0, 9] = float("nan"), float("inf")
            c.append([0], [172], k, v)
            q = c.randn(rows, 2, 64)
            out = torch.empty_like(q)
            D.q8_attend(c.cache, q, out, ints([172]))
            seen = 172 - (rows - 1) + torch.arange(rows, device="cuda")
            for dim, t, what in ((7, 169, torch.isnan), (9, 170, torch.isinf)):
                assert torch.equal(what(out[:, :, dim]), (seen > t)[:, None].expand(rows, 2))
            keep = [d for d in range(64) if d not in (7, 9)]
            assert torch.isfinite(out[:, :, keep]).all()


@pytest.mark.parametrize("rows", [1, 140])
def test_empty_sequences_and_bad_ones_among_many_rows(rows):
    for dtype in (F32, BF16):
        c = Case(4, 2, 192, 64, "e4m3", dtype, seed=4)
        c.append([0, 1, 2, 3], [190, 3, 20, 160])
        q = c.randn(5 * rows, 4, 64)
        out, status = torch.full_like(q, 77.0), ints([0])
        D.q8_attend(c.cache, q, out, ints([190, 0, 193, 20, 160]), slots=ints([0, 1, 2, -1, 9]), status=status)
        out = out.view(5, rows, 4, 64)
        assert torch.isfinite(out[0]).all() and (out[1] == 0).all() and torch.isnan(out[2]).all()
        assert (out[3] == 77.0).all() and torch.isnan(out[4]).all() and status.item() == 1


@pytest.mark.parametrize("rows", [1, 3, 70, 160])
def test_a_sequence_does_not_depend_on_the_batch(rows):
    c = Case(40, 2, 3088, 64, "int8", BF16, seed=rows)
    lens = [3000 if i == 7 else 160 + 3 * i for i in range(40)]
    c.append(list(range(40)), lens)
    q = c.randn(40 * rows, 8, 64)
    every = torch.empty_like(q)
    D.q8_attend(c.cache, q, every, ints(lens))
    for i in (0, 7, 39):
        one = torch.empty_like(q[:rows])
        for most in (0, lens[i]):
            D.q8_attend(c.cache, q[i * rows:(i + 1) * rows], one, ints([lens[i]]), slots=ints([i]), max_len=most)
            assert torch.equal(one, every[i * rows:(i + 1) * rows])


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F32), (256, F16)])
def test_long_sequences_and_their_workspace(hd, dtype):
    """More splits than a cluster holds: results through the workspace, and the same ones in any batch."""
    longest = 20100 if hd == 64 else 11001
    c = Case(3, 1, longest + 15 & ~15, hd, "int8", dtype, seed=hd)
    lens = [longest, 700, longest - 1500]
    c.append([0, 1, 2], lens)
    for rows in (1, 2):
        out = c.attend_check([0, 1, 2], [rows] * 3, 4)
        q = c.randn(3 * rows, 4, hd)
        D.q8_attend(c.cache, q, out, ints(lens))
        for i in range(3):
            one = torch.empty_like(q[:rows])
            need = D.q8.workspace_bytes(c.cache, rows, 4, lens[i])
            assert (need > 0) == (lens[i] > 9000)
            ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
            D.q8_attend(c.cache, q[i * rows:(i + 1) * rows], one, ints([lens[i]]), slots=ints([i]), max_len=lens[i],
                        workspace=ws)
            assert torch.equal(one, out[i * rows:(i + 1) * rows])
        with pytest.raises(D.InvalidArgumentError, match="workspace"):
            D.q8_attend(c.cache, q, out, ints(lens), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    # from another stream, and a max_len that is too small: still whole sequences
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    two = torch.empty_like(out)
    D.q8_attend(c.cache, q, two, ints(lens), stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(out, two)
    c.attend_check([0, 1, 2], [1] * 3, 4, max_len=16)


def test_strided_queries_and_outputs():
    for rows in (1, 90):
        c = Case(2, 2, 128, 64, "int8", F16)
        c.append([0, 1], [100, 121])
        q = c.randn(2 * rows, 4, 64)
        want = torch.empty_like(q)
        D.q8_attend(c.cache, q, want, ints([100, 121]))
        qq = torch.zeros(4, 2 * rows, 67, dtype=F16, device="cuda")
        qq[:, :, 3:] = q.transpose(0, 1)
        out = torch.full((2 * rows, 5, 65), 7.0, dtype=F16, device="cuda")
        D.q8_attend(c.cache, qq[:, :, 3:].transpose(0, 1), out[:, :4, 1:], ints([100, 121]))
        assert torch.equal(out[:, :4, 1:], want)
        assert (out[:, 4] == 7.0).all() and (out[:, :, 0] == 7.0).all()


def test_streams_and_graphs():
    """A captured decode step (append, attend, read) replayed with new contents, on a stream of its own."""
    c = Case(3, 2, 96, 64, "int8", BF16)
    c.append([0, 1, 2], [14, 31, 40])
    st = torch.cuda.Stream()
    k, v, q = torch.empty(3, 2, 64, dtype=BF16, device="cuda"), torch.empty(3, 2, 64, dtype=BF16, device="cuda"), \
        torch.empty(3, 4, 64, dtype=BF16, device="cuda")
    out = torch.empty_like(q)
    pos, lens = ints([14, 31, 40]), ints([15, 32, 41])
    back = [torch.zeros(3, 2, 96, 64, dtype=BF16, device="cuda") for _ in range(2)]

    def step():
        D.q8_append(c.cache, k, v, pos)
        D.q8_attend(c.cache, q, out, lens)
        D.q8_read(c.cache, *back, lens)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        step()
    for _ in range(20):
        nk, nv, nq = c.randn(3, 2, 64), c.randn(3, 2, 64), c.randn(3, 4, 64)
        k.copy_(nk), v.copy_(nv), q.copy_(nq)
        for s in range(3):
            c.plain[s][0].append(nk[s:s + 1])
            c.plain[s][1].append(nv[s:s + 1])
        g.replay()
        pos += 1
        lens += 1
        torch.cuda.synchronize()
        for s in range(3):
            kk, vv = c.values(s)
            want, most = attend64(nq[s:s + 1].double().cpu().numpy(), kk, vv, [c.len(s)], None, 64 ** -0.5)
            assert far(out[s:s + 1], want) <= tolerance(BF16, most)
            w = torch.tensor(kk.astype(np.float32), device="cuda").to(BF16)
            assert torch.equal(back[0][s, :, :c.len(s)], w)
    c.check()
    # the default argument follows torch's current stream; an explicit one is taken as it is
    a, b = torch.empty_like(q), torch.empty_like(q)
    with torch.cuda.stream(st):
        D.q8_attend(c.cache, q, a, lens)
    st.synchronize()
    D.q8_attend(c.cache, q, b, lens, stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(a, b)


def test_two_calls_at_once():
    """Long sequences on two streams, each with a workspace of its own, and two replayed graphs."""
    c = Case(2, 2, 12016, 128, "int8", BF16, seed=6)
    c.append([0, 1], [12000, 9990])
    q = [c.randn(2, 8, 128) for _ in range(2)]
    want = [D.q8_attend(c.cache, x, torch.empty_like(x), ints([12000, 9990])).clone() for x in q]
    torch.cuda.synchronize()
    lens = ints([12000, 9990])
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(x) for x in q]
    graphs = []
    for x, o, s in zip(q, outs, st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            D.q8_attend(c.cache, x, o, lens)
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, st):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
    for _ in range(5):
        for x, o, s in zip(q, outs, st):
            o.zero_()
            s.wait_stream(torch.cuda.current_stream())
            D.q8_attend(c.cache, x, o, lens, stream=s.cuda_stream)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """A slot behind 4 GB of codes, and a position whose codes lie 4 GB into its head."""
    n = 1 << 24
    cap, hd = n + 64, 256
    g = torch.Generator("cuda").manual_seed(0)
    codes = [torch.empty(2, 1, cap, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(2, 1, cap // 16, device="cuda") for _ in range(2)]
    tails = [torch.zeros(2, 1, 16, hd, dtype=BF16, device="cuda") for _ in range(2)]
    cache = D.Q8Cache(*codes, *scales, *tails)
    k, v = (torch.randn(40, 1, hd, device="cuda", generator=g).to(BF16) for _ in range(2))
    D.q8_append(cache, k, v, ints([n]), slots=ints([1]))
    twin = Case(1, 1, 64, hd, "int8", BF16)
    twin.append([0], [40], k, v)
    back = [torch.zeros(1, 1, 40, hd, dtype=BF16, device="cuda") for _ in range(2)]
    D.q8_read(cache, *back, ints([n + 40]), start=ints([n]), slots=ints([1]))
    for got, want in zip(back, twin.values(0)):
        assert torch.equal(got[0], torch.tensor(want.astype(np.float32), device="cuda").to(BF16))
    # the positions before those are hidden: codes and scales of any value, as long as they are numbers
    for x in codes:
        x[1, 0, :n] = 1
    for x in scales:
        x[1, 0, :n // 16] = 1.0
    masked = torch.zeros(1, cap, dtype=torch.uint8, device="cuda")
    masked[0, :n] = 1
    for rows in (1, 80):
        q = torch.randn(rows, 2, hd, device="cuda", generator=g).to(BF16)
        out = torch.empty_like(q)
        D.q8_attend(cache, q, out, ints([n + 40]), slots=ints([1]), masked=masked, causal=False)
        want, most = attend64(q.double().cpu().numpy(), *twin.values(0), [40] * rows, None, hd ** -0.5)
        assert far(out, want) <= tolerance(BF16, most)


def test_generation_together():
    """A prompt, then single tokens: every step's attention against 64 bits."""
    for kind in ("int8", "e4m3"):
        c = Case(2, 2, 96, 64, kind, F32, seed=5)
        c.append([0, 1], [37, 12])
        c.attend_check([0, 1], [37, 12], 6)
        for _ in range(30):
            c.append([1, 0], [1, 1])
            c.attend_check([1, 0], [1, 1], 6)
        c.check()
