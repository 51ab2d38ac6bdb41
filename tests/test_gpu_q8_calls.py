"""8-bit key/value cache on the GPU: calls that the documentation allows beside
the ordinary ones (launch sizes, threads, streams, workspaces)."""
import os
import subprocess
import sys

import pytest

import defer_b200 as D
from tests.conftest import ROOT
from tests.test_gpu_q8 import Case, ints
from tests.test_gpu_q8_values import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length", [0, 20, 300, 1100])
@pytest.mark.parametrize("causal", [True, False])
def test_a_max_q_below_the_rows(dtype, hd, length, causal):
    """A CTA then takes many tiles, the first ones of which see nothing when there are more rows than positions."""
    rows = 1000
    c = Case(2, 1, 1104, hd, "int8", dtype, seed=length)
    c.append([0, 1], [length, 40])
    start = ints([0, rows, 2 * rows])
    for max_q in (40, 200):
        check(c, [0, 1], rows, 2, causal=causal, q_start=start, max_q=max_q)


FIRST_CALLS = """
import threading
import torch
import defer_b200 as D

refused = []
torch.zeros(1, device="cuda")

def first_call(kind, dtype, hd, rows, start):
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        z = lambda *s, dt: torch.zeros(*s, dtype=dt, device="cuda")
        c = D.Q8Cache(z(1, 1, 32, hd, dt=kind), z(1, 1, 32, hd, dt=kind), z(1, 1, 2, dt=torch.float32),
                      z(1, 1, 2, dt=torch.float32), z(1, 1, 16, hd, dt=dtype), z(1, 1, 16, hd, dt=dtype))
        q = z(rows, 1, hd, dt=dtype)
        out = torch.empty_like(q)
        lens = torch.full((1,), 5, dtype=torch.int32, device="cuda")
        st.synchronize()
        start.wait()
        try:
            D.q8_attend(c, q, out, lens)
        except D.DeferError as e:
            refused.append((str(kind), hd, rows, str(e)))
        st.synchronize()

# kernels that need more shared memory than a launch gets unasked
for kind in (torch.int8, torch.float8_e4m3fn):
    for dtype, hd, rows in ((torch.float32, 256, 1), (torch.float32, 128, 12), (torch.float32, 80, 12),
                            (torch.bfloat16, 128, 100), (torch.bfloat16, 64, 100)):
        start = threading.Barrier(8)
        ts = [threading.Thread(target=first_call, args=(kind, dtype, hd, rows, start)) for _ in range(8)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
print(refused)
assert not refused
"""


def test_first_calls_of_several_threads():
    """A process of its own, whose threads make their first calls at the same moment."""
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT},
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout + r.stderr[-2000:]


def test_a_workspace_of_the_size_that_is_named():
    """64 sequences of one row, and ragged ones, over more than one cluster's splits."""
    n, length = 64, 9600
    c = Case(n, 2, length, 128, "int8", BF16)
    for x in c.codes:
        x.zero_()
    for x in (*c.scales, *c.tails):
        x.zero_()
    q = c.randn(n, 16, 128)
    lens = ints([length - 150 * i for i in range(n)])
    need = D.q8.workspace_bytes(c.cache, n, 16, length)
    assert need
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 77.0)
    D.q8_attend(c.cache, q, out, lens, max_len=length, workspace=ws)
    assert (out == 0).all()  # the values are zeros
    out.fill_(77.0)
    D.q8_attend(c.cache, q, out, lens[:3].contiguous(), q_start=ints([0, 1, 40, n]), slots=ints([5, 6, 7]), max_q=39,
                max_len=length, workspace=ws)
    assert (out == 0).all()
    with pytest.raises(D.InvalidArgumentError, match="workspace"):
        D.q8_attend(c.cache, q, out, lens, max_len=length, workspace=ws[:need - 16])


@pytest.mark.parametrize("other", ["default", "stream"])
def test_the_workspace_belongs_to_the_calls_stream(other):
    """A call on a stream that is not torch's current one: its workspace goes back to that stream's memory."""
    target = torch.cuda.default_stream() if other == "default" else torch.cuda.Stream()
    size = 48 << 20
    with torch.cuda.stream(torch.cuda.Stream()):
        ws = D.q8._scratch(0, size, target.cuda_stream)
        at = ws.data_ptr()
        del ws
        mine = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert mine.data_ptr() != at
    with torch.cuda.stream(target):
        assert torch.empty(size, dtype=torch.uint8, device="cuda").data_ptr() == at
