"""8-bit key/value cache: what the Python calls turn away and promise, without a GPU."""
import pytest

import defer_b200 as D
from defer_b200 import q8

P = 0x10000  # a non-null, aligned address that nothing may touch


class Array:
    """An array that is on no device: what the checks look at."""
    is_cuda = True

    def __init__(self, *shape, dtype="torch.float32"):
        self.shape, self.dtype = shape, dtype

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def stride(self, d=None):
        st, n = [], 1
        for x in reversed(self.shape):
            st.insert(0, n)
            n *= x
        return tuple(st) if d is None else st[d]

    def data_ptr(self):
        return P


def cache(slots=4, kvh=2, cap=64, hd=64, kind="torch.int8", dtype="torch.float32"):
    c, s, t = Array(slots, kvh, cap, hd, dtype=kind), Array(slots, kvh, cap // 16), Array(slots, kvh, 16, hd, dtype=dtype)
    return D.Q8Cache(c, c, s, s, t, t)


def ints(n):
    return Array(n, dtype="torch.int32")


@pytest.mark.parametrize("dtype", ["torch.float32", "torch.bfloat16", "torch.float16"])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("length", [4096, 9216, 16384, 65536, 1 << 20])
def test_workspace_bytes_serves_every_batch(dtype, hd, length):
    c = cache(slots=64, kvh=8, cap=1 << 20, hd=hd, dtype=dtype)
    for tokens in (1, 4, 64, 512):
        most = q8.workspace_bytes(c, tokens, 32, length)
        assert (most > 0) == (length >= {32: 36864, 64: 18432}.get(hd, 9216))
        for n in (1, 2, 64):
            if tokens % n == 0:
                need = q8._workspace_bytes(c, q8._batch(0, n, tokens, 0, None, None, None), length, 32)
                assert need <= most and need == q8.workspace_bytes(c, tokens, 32, length, n=n)
        for max_q in (0, 1, 16, 64):
            assert q8._workspace_bytes(c, q8._batch(0, 3, tokens, max_q, ints(4), None, None), length, 32) <= most


@pytest.mark.parametrize("bad", [-1, 1 << 32, (1 << 32) + 5])
def test_counts_out_of_range_are_refused(bad):
    c, kv, q = cache(), Array(4, 2, 64), Array(4, 4, 64)
    for call in (lambda: D.q8_append(c, kv, kv, ints(4), max_q=bad), lambda: D.q8_attend(c, q, q, ints(4), max_q=bad),
                 lambda: D.q8_attend(c, q, q, ints(4), max_len=bad), lambda: q8.workspace_bytes(c, bad, 4),
                 lambda: q8.workspace_bytes(c, 4, bad), lambda: q8.workspace_bytes(c, 4, 4, bad),
                 lambda: q8.workspace_bytes(c, 4, 4, n=bad)):
        with pytest.raises(D.InvalidArgumentError, match="2\\^32"):
            call()


def test_what_is_no_cache_is_refused():
    q = Array(4, 4, 64)
    for call in (lambda: D.q8_append(None, q, q, ints(4)), lambda: D.q8_attend(q, q, q, ints(4)),
                 lambda: D.q8_read("layer", q, q, ints(4)), lambda: q8.workspace_bytes(object(), 4, 4)):
        with pytest.raises(D.InvalidArgumentError, match="Q8Cache"):
            call()


@pytest.mark.parametrize("role,wait_us", [(0, 1000), (6, 1000), (-1, 1000), (2, 0), (2, 10 ** 6 + 1)])
def test_drill_refusals(role, wait_us):
    with pytest.raises(D.InvalidArgumentError):
        q8.stall_next_attend(role, wait_us)


def test_an_append_of_too_many_slots_is_refused():
    """Its search for a slot that is named twice grows with the square of them."""
    n = (1 << 16) + 1
    c, kv = cache(slots=1 << 20, kvh=1, cap=16, hd=16), Array(n, 1, 16)
    with pytest.raises(D.InvalidArgumentError, match="slots"):
        D.q8_append(c, kv, kv, ints(n), slots=ints(n), stream=0)
