"""A layer of a model's 8-bit caches under the operators (QuantKvCache.view)."""
import gc

import numpy as np
import pytest

import defer_b200 as D
from tests.gpu_util import model_file
from tests.q8_util import attend64, far, tolerance

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_operators_on_a_layers_view(tmp_path, kind):
    m = D.Model.load(model_file(str(tmp_path), "test-gqa4"))
    c = m.config
    qc = m.new_quant_cache(2, 48, kind)
    for t in range(37):
        m.forward_q8([t, t + 1], qc)
    view = qc.view(1)
    want = [x.reshape(37, c.num_kv_heads, c.head_dim).transpose(1, 0, 2) for x in qc.layer(1, 1)]
    k, v = (torch.zeros(1, c.num_kv_heads, 37, c.head_dim, device="cuda") for _ in range(2))
    D.q8_read(view, k, v, ints([37]), slots=ints([1]))
    for got, x in zip((k, v), want):
        assert np.array_equal(got[0].cpu().numpy(), x)
    g = torch.Generator("cuda").manual_seed(0)
    q = torch.randn(3, c.num_heads, c.head_dim, device="cuda", generator=g)
    out = D.q8_attend(view, q, torch.empty_like(q), ints([37]), slots=ints([1]))
    ref, most = attend64(q.double().cpu().numpy(), *(x.astype(np.float64) for x in want), [35, 36, 37], None,
                         c.head_dim ** -0.5)
    assert far(out, ref) <= tolerance(torch.float32, most)
    rows = torch.randn(2, c.num_kv_heads, c.head_dim, device="cuda", generator=g)
    D.q8_append(view, rows, rows, ints([37]), slots=ints([1]))
    D.q8_read(view, k[:, :, :2], v[:, :, :2], ints([39]), start=ints([37]), slots=ints([1]))
    assert torch.equal(k[0, :, :2], rows.transpose(0, 1)) and torch.equal(v[0, :, :2], rows.transpose(0, 1))
    assert D.q8.workspace_bytes(view, 1, c.num_heads) == 0
    with pytest.raises(D.InvalidArgumentError, match="float32"):
        D.q8_attend(view, q.half(), torch.empty_like(q.half()), ints([37]), slots=ints([1]))


def test_a_view_keeps_its_cache(tmp_path):
    m = D.Model.load(model_file(str(tmp_path), "test-gqa4"))
    qc = m.new_quant_cache(1, 16)
    m.forward_q8([3], qc)
    want = qc.layer(0)[0]
    view = qc.view(0)
    del qc
    gc.collect()
    assert view.owner.len(0) == 1
    k, v = (torch.zeros(1, m.config.num_kv_heads, 1, m.config.head_dim, device="cuda") for _ in range(2))
    D.q8_read(view, k, v, ints([1]))
    assert np.array_equal(k.cpu().numpy().ravel(), want)
