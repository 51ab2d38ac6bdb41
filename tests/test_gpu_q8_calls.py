"""8-bit key/value cache on the GPU: calls that the documentation allows beside
the ordinary ones (launch sizes, threads, streams, workspaces)."""
import pytest

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
