"""8-bit key/value cache: refusals, without a GPU. Every call here must be
turned away by the host's checks before anything is launched."""
import ctypes
import struct

import pytest

import defer_b200 as D
from defer_b200 import _lib

P = 0x10000  # a non-null, aligned address that nothing may touch


def cache(**kw):
    c = _lib.Q8CacheC(0, 0, 0, 4, 2, 64, 64, P, P, P, P, P, P)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(n=2, tokens=2):
    return struct.pack("=IIIxxxxQQQ", n, tokens, 0, 0, 0, 0)


def attend(c=None, b=None, lens=P, heads=4, q=P, out=P, ot=256, oh=64, masked=None, ms=0, scale=0.125):
    c, b = c or cache(), b or batch()
    return _lib.load().defer_q8_attend(ctypes.addressof(c), b, lens, 0, heads, q, 256, 64, out, ot,
                                       oh, masked, ms, 1, scale, None, 0, None)


def append(c=None, b=None, pos=P, k=P, v=P):
    c, b = c or cache(), b or batch()
    return _lib.load().defer_q8_append(ctypes.addressof(c), b, pos, k, 128, 64, v, 128, 64, None)


def read(c=None, n=2, lens=P, rows=8, ko=P, ks=(1024, 512, 64), vs=(1024, 512, 64)):
    c = c or cache()
    return _lib.load().defer_q8_read(ctypes.addressof(c), n, lens, None, None, None, rows, ko, struct.pack("=qqq", *ks), P,
                                      struct.pack("=qqq", *vs), None)


BAD = D.InvalidArgumentError.code


@pytest.mark.parametrize("field,value", [
    ("k_codes", 0), ("v_scales", 0), ("v_tail", P + 8), ("kind", 2), ("kind", -1), ("dtype", 3), ("slots", 0),
    ("kv_heads", 0), ("cap", 0), ("cap", 24), ("head_dim", 0), ("head_dim", 24), ("head_dim", 272), ("device", -1)])
def test_a_bad_cache_is_refused(field, value):
    for call in (attend, append, read):
        assert call(cache(**{field: value})) == BAD
        assert _lib.load().defer_last_error()


def test_null_descriptors_are_refused():
    L = _lib.load()
    b = batch()
    assert L.defer_q8_append(None, b, P, P, 128, 64, P, 128, 64, None) == BAD
    c = cache()
    assert L.defer_q8_append(ctypes.addressof(c), None, P, P, 128, 64, P, 128, 64, None) == BAD


@pytest.mark.parametrize("kw", [dict(b=batch(tokens=3)), dict(b=batch(n=5, tokens=5)), dict(b=batch(n=0)), dict(lens=None),
                                dict(heads=3), dict(heads=0), dict(q=None), dict(out=None), dict(ot=192), dict(oh=32),
                                dict(masked=P, ms=63), dict(scale=float("nan")), dict(scale=float("inf")),
                                dict(b=batch(n=4, tokens=1 << 29), heads=4)])
def test_attend_refusals(kw):
    assert attend(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(b=batch(tokens=3)), dict(b=batch(n=5, tokens=5)), dict(pos=None), dict(k=None),
                                dict(v=None)])
def test_append_refusals(kw):
    assert append(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(n=5), dict(lens=None), dict(ko=None), dict(ks=(1024, 512, 32)),
                                dict(ks=(512, 512, 64)), dict(vs=(1024, 64, 64))])
def test_read_refusals(kw):
    assert read(**kw) == BAD


def test_empty_calls_do_nothing():
    assert attend(b=batch(n=0, tokens=0)) == 0
    assert append(b=batch(n=2, tokens=0)) == 0
    assert read(n=0) == 0 and read(rows=0) == 0


def test_python_checks():
    torch = pytest.importorskip("torch")
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)  # noqa: E731
    good = [z(2, 2, 32, 64, dt=torch.int8), z(2, 2, 32, 64, dt=torch.int8), z(2, 2, 2), z(2, 2, 2), z(2, 2, 16, 64),
            z(2, 2, 16, 64)]
    with pytest.raises(D.InvalidArgumentError, match="CUDA"):  # host memory
        D.Q8Cache(*good)
    for i, x in ((0, z(2, 2, 32, 64)), (1, z(2, 2, 16, 64, dt=torch.int8)), (2, z(2, 2, 3)), (3, z(2, 2, 2).double()),
                 (4, z(2, 2, 15, 64)), (5, z(2, 2, 16, 64).half()), (0, z(2, 32, 64, dt=torch.int8)),
                 (0, z(2, 2, 40, 64, dt=torch.int8))):
        with pytest.raises(D.InvalidArgumentError):
            D.Q8Cache(*[x if j == i else y for j, y in enumerate(good)])
