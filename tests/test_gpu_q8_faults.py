"""The tile kernel's bounded waits, made to run out from the host: one role of
the kernel withholds its arrivals with the waits cut to a millisecond. The
kernel returns by itself, its rows are NaN, the status word says so, and the
next call is unaffected. Nothing faults, traps or hangs."""
import pytest

import defer_b200 as D
from tests.test_gpu_q8 import Case, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("role", [1, 2, 3, 4, 5])
def test_a_role_that_does_not_arrive(dtype, hd, role):
    rows = [300, 5, 140]  # tiles, the streaming kernel's, tiles
    c = Case(3, 1, 720, hd, "int8", dtype, seed=role)
    c.append([0, 1, 2], [705, 100, 13])  # many blocks, and open blocks alone
    q = c.randn(sum(rows) + 2, 4, hd)
    lens, start = ints([705, 100, 13]), ints([0, 300, 305, 445])

    def call():
        out, status = torch.full_like(q, 77.0), ints([0])
        D.q8_attend(c.cache, q, out, lens, q_start=start, max_q=300, causal=False, status=status)
        return out, status.item()

    want, status = call()
    assert status == 0 and torch.isfinite(want).all()
    D.q8.stall_next_attend(role, 1000)
    out, status = call()
    assert status == 4
    assert torch.isnan(out[:300]).all() and torch.isnan(out[305:445]).all()
    assert torch.equal(out[300:305], want[300:305]) and (out[445:] == 77.0).all()
    out, status = call()
    assert status == 0 and torch.equal(out, want)


def test_a_cta_of_several_tiles_gives_up_once():
    c = Case(1, 1, 320, 64, "int8", torch.bfloat16)
    c.append([0], [301])
    q = c.randn(1000, 2, 64)
    for role in (1, 2, 3, 4, 5):
        out, status = torch.full_like(q, 77.0), ints([0])
        D.q8.stall_next_attend(role, 1000)
        D.q8_attend(c.cache, q, out, ints([301]), q_start=ints([0, 1000]), max_q=40, causal=False, status=status)
        assert status.item() == 4 and torch.isnan(out).all()
