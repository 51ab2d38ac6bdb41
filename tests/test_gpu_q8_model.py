"""A model's step over an 8-bit cache (Model.forward_q8) and the conversions
between KvCache and QuantKvCache.

The step is checked against the fp32 one on the same values: the 8-bit slot is
read back into a KvCache, and Model.forward of the next token on that cache
must give the same logits at the parity tolerance, as long as the token does
not close a block (its own row would be quantised before the attention)."""
import ctypes
import struct

import numpy as np
import pytest

import defer_b200 as D
from defer_b200 import _lib, synthetic
from tests.gpu_util import logits_close, model_file
from tests.q8_util import quantise

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def shape_file(directory, name):
    if name != "wide-bf16":
        return model_file(directory, name)
    # bf16 and hidden >= 2048: the token loops of this model run on the tensor cores
    s = synthetic.Shape(1000, 2048, 1024, 2, 16, 4, 128, 10000.0, False, max_position_embeddings=256, bf16=True)
    return synthetic.write_normal_model(f"{directory}/wide.safetensors", s)


@pytest.mark.parametrize("name", ["tiny", "test-gqa4", "test-bf16", "wide-bf16"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_step_matches_the_fp32_step_on_the_same_values(tmp_path, name, kind):
    m = D.Model.load(shape_file(str(tmp_path), name))
    c = m.config
    qc = m.new_quant_cache(3, 80, kind)
    toks = [int(t) for t in np.random.default_rng(1).integers(0, c.vocab_size, 70)]
    full = m.new_cache(96)
    for pos, t in enumerate(toks):
        want = m.forward(t, qc.load(1)) if (pos + 1) % 16 else None
        got = m.forward_q8([t], qc, [1])[0]
        plain = m.forward(t, full)
        assert qc.len(1) == pos + 1 and qc.len(0) == qc.len(2) == 0
        if want is not None:
            ok, err, rng = logits_close(got, want)
            assert ok, (pos, err, rng)
        # and near the all-fp32 model: a cache value is off by half a step, 1/254 (2^-4 of itself for e4m3) at most
        assert np.abs(got - plain).max() <= 0.2 * (plain.max() - plain.min()), pos
    # layer 0's rows depend on the tokens alone: the stored values are the definition's
    kq, vq = (x.reshape(70, c.num_kv_heads, c.head_dim) for x in qc.layer(0, 1))
    kf, vf = (x.reshape(70, c.num_kv_heads, c.head_dim) for x in full.layer(0))
    for got, x in ((kq, kf), (vq, vf)):
        for h in range(c.num_kv_heads):
            for b in range(4):
                code, s = quantise(x[16 * b:16 * b + 16, h], kind)
                assert np.array_equal(got[16 * b:16 * b + 16, h], (code.astype(np.float32) * s))
        assert np.array_equal(got[64:], x[64:])


@pytest.mark.parametrize("name", ["test-gqa4", "wide-bf16"])
def test_slots_do_not_depend_on_each_other(tmp_path, name):
    m = D.Model.load(shape_file(str(tmp_path), name))
    r = np.random.default_rng(2)
    lens = [1, 16, 40, 5, 33, 17, 2, 29, 12, 31]
    toks = [[int(t) for t in r.integers(0, m.config.vocab_size, n)] for n in lens]
    together = m.new_quant_cache(12, 64)
    last = {}
    for step in range(max(lens)):
        live = [i for i, n in enumerate(lens) if step < n]
        out = m.forward_q8([toks[i][step] for i in live], together, [i + 1 for i in live])
        last.update({i: out[j] for j, i in enumerate(live)})
    for i, n in enumerate(lens):
        alone = m.new_quant_cache(1, 64)
        for t in toks[i]:
            out = m.forward_q8([t], alone)
        assert np.array_equal(out[0].view(np.uint32), last[i].view(np.uint32)), i
        for l in range(m.config.num_layers):
            for a, b in zip(alone.layer(l), together.layer(l, i + 1)):
                assert np.array_equal(a, b)


def test_store_load_and_truncate(tmp_path):
    m = D.Model.load(model_file(str(tmp_path), "test-gqa4"))
    c = m.config
    r = np.random.default_rng(3)
    toks = [int(t) for t in r.integers(0, c.vocab_size, 45)]
    full = m.new_cache(64)
    for t in toks:
        m.forward(t, full)
    qc = m.new_quant_cache(2, 64)
    qc.store(full, 1)
    assert qc.len(1) == 45 and qc.len(0) == 0
    for l in range(c.num_layers):
        for got, x in zip(qc.layer(l, 1), full.layer(l)):
            got, x = (y.reshape(45, c.num_kv_heads, c.head_dim) for y in (got, x))
            for h in range(c.num_kv_heads):
                for b in range(2):
                    code, s = quantise(x[16 * b:16 * b + 16, h], "int8")
                    assert np.array_equal(got[16 * b:16 * b + 16, h], code.astype(np.float32) * s)
            assert np.array_equal(got[32:], x[32:])
    back = qc.load(1)
    assert len(back) == 45
    for l in range(c.num_layers):
        for a, b in zip(back.layer(l), qc.layer(l, 1)):
            assert np.array_equal(a, b)
    # the stored cache goes on like the one it came from
    ok, err, rng = logits_close(m.forward_q8([7], qc, [1])[0], m.forward(7, back))
    assert ok, (err, rng)
    # shortened inside the open block, into a closed one, to a border
    for n in (41, 21, 16, 3, 0):
        was = [qc.layer(l, 1) for l in range(c.num_layers)]
        qc.truncate(n, 1)
        assert qc.len(1) == n
        for l in range(c.num_layers):
            for a, b in zip(qc.layer(l, 1), was[l]):
                assert np.array_equal(a, b[:n * c.kv_dim])
        if n:
            want = m.forward(9, qc.load(1))
            ok, err, rng = logits_close(m.forward_q8([9], qc, [1])[0], want)
            assert ok, (n, err, rng)
            qc.truncate(n, 1)
    qc.truncate(5, 1)
    assert qc.len(1) == 0


def test_refusals(tmp_path):
    m = D.Model.load(model_file(str(tmp_path), "tiny"))
    other = D.Model.load(model_file(str(tmp_path), "test-gqa4"))
    qc = m.new_quant_cache(2, 17)
    for bad in (lambda: m.new_quant_cache(0), lambda: m.new_quant_cache(1, 16, "int4"),
                lambda: m.forward_q8([1, 2], qc, [0, 0]), lambda: m.forward_q8([1], qc, [2]),
                lambda: m.forward_q8([1, 2, 3], qc), lambda: m.forward_q8([1], qc, [0, 1]),
                lambda: other.forward_q8([1], qc), lambda: qc.load(2), lambda: qc.truncate(0, 5),
                lambda: qc.store(other.new_cache(16)), lambda: qc.view(2), lambda: qc.layer(9)):
        with pytest.raises(D.InvalidArgumentError):
            bad()
    with pytest.raises(D.ModelError, match="out of range"):
        m.forward_q8([m.config.vocab_size], qc)
    big = m.new_cache(64)
    for _ in range(33):
        m.forward(1, big)
    with pytest.raises(D.ModelError, match="capacity"):
        qc.store(big)
    for _ in range(32):  # 17 positions were rounded up to 32
        m.forward_q8([5, 6], qc)
    with pytest.raises(D.ModelError, match="capacity"):
        m.forward_q8([5], qc, [1])
    assert qc.len(0) == qc.len(1) == 32
    assert m.forward_q8([], qc).shape == (0, m.config.vocab_size)


def test_a_layers_view_serves_the_operators(tmp_path):
    m = D.Model.load(model_file(str(tmp_path), "test-bf16"))
    c = m.config
    qc = m.new_quant_cache(2, 48, "e4m3")
    for t in range(37):
        m.forward_q8([t, t + 1], qc)
    v = qc.view(1)
    k, w = (torch.zeros(1, c.num_kv_heads, 37, c.head_dim, device="cuda") for _ in range(2))
    lens, slots = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (37, 1))
    st = struct.pack("=qqq", *k.stride()[:3])
    rc = _lib.load().defer_q8_read(ctypes.addressof(v), 1, lens.data_ptr(), None, slots.data_ptr(), None, 37,
                                   k.data_ptr(), st, w.data_ptr(), st, None)
    torch.cuda.synchronize()
    assert rc == 0
    for got, want in zip((k, w), qc.layer(1, 1)):
        assert np.array_equal(got[0].cpu().numpy(), want.reshape(37, c.num_kv_heads, c.head_dim).transpose(1, 0, 2))


def test_greedy_generation_stays_near_the_fp32_model(tmp_path):
    """The steps of several sessions together, each choosing its own tokens."""
    m = D.Model.load(model_file(str(tmp_path), "test-gqa4"))
    prompts = [[3, 5, 8], [400, 2, 77, 61, 9]]
    qc = m.new_quant_cache(2, 64)
    logits = [None, None]
    for i, p in enumerate(prompts):
        for t in p:
            logits[i] = m.forward_q8([t], qc, [i])[0]
    for _ in range(24):
        toks = [D.sample_logits(x, 0.0)[0] for x in logits]
        wants = [m.forward(t, qc.load(i)) for i, t in enumerate(toks)]
        logits = list(m.forward_q8(toks, qc))
        for i in range(2):
            if qc.len(i) % 16:
                ok, err, rng = logits_close(logits[i], wants[i])
                assert ok, (i, err, rng)


