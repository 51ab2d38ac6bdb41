"""Model.forward_q8 of more slots than a tensor-core step has (128)."""
import numpy as np
import pytest

import defer_b200 as D
from tests.test_gpu_q8_model import shape_file

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["wide-bf16", "test-gqa4"])
def test_more_slots_than_one_step(tmp_path, name):
    m = D.Model.load(shape_file(str(tmp_path), name))
    n = 131
    toks = np.random.default_rng(4).integers(0, m.config.vocab_size, (3, n))
    together, alone = m.new_quant_cache(n, 16), m.new_quant_cache(n, 16)
    order = [(7 * i) % n for i in range(n)]
    for step in range(3):
        got = m.forward_q8([int(toks[step, s]) for s in order], together, order)
        assert got.shape == (n, m.config.vocab_size)
        for i in (0, 127, 128, 130):
            s = order[i]
            want = m.forward_q8([int(toks[step, s])], alone, [s])[0]
            assert np.array_equal(got[i].view(np.uint32), want.view(np.uint32)), (step, i)
    assert all(together.len(s) == 3 for s in range(n))
    for s in (order[128], order[0]):
        for a, b in zip(together.layer(1, s), alone.layer(1, s)):
            assert np.array_equal(a, b)
