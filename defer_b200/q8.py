"""Key/value cache in 8 bits on the caller's device buffers: defer_q8_append,
defer_q8_read and defer_q8_attend of include/defer_b200.h for arrays that
have a device pointer (torch CUDA tensors; torch itself is not imported).

    cache = Q8Cache(k_codes, v_codes, k_scales, v_scales, k_tail, v_tail)
    q8_append(cache, k, v, pos)             # rows into the cache
    q8_attend(cache, q, out, lens)          # attention over it
    q8_read(cache, k_out, v_out, lens)      # values back

Every call launches on `stream` (a cudaStream_t as an integer), by default
torch's current stream of the cache's device, and waits for nothing, so it may
be captured into a CUDA graph (make one such call before the capture: CUDA
loads device code at a kernel's first launch). Nothing is allocated on the
device but the workspace of long sequences (q8_attend). The arrays must stay
allocated until the stream has run the call.
"""
from __future__ import annotations

import ctypes
import struct
import sys
from typing import Optional

from . import _lib

BLOCK = 16  # positions that share a scale
_DTYPES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2}
_KINDS = {"torch.int8": 0, "torch.float8_e4m3fn": 1}
_BYTES = ("torch.uint8", "torch.bool", "torch.int8")
_BATCH = struct.Struct("=IIIxxxxQQQ")  # defer_q8_batch
_STRIDES = struct.Struct("=qqq")
_check = None  # the package's status check (set by defer_b200/__init__.py)
_invalid = None


def _refuse(what: str):
    raise _invalid("8-bit cache: " + what)


def _stream_of(device: int) -> int:
    t = sys.modules.get("torch")
    if t is None:
        return 0
    raw = getattr(t._C, "_cuda_getCurrentRawStream", None)  # a tenth of the public call's time
    return raw(device) if raw is not None else t.cuda.current_stream(device).cuda_stream


_names = {}  # dtype object -> its name (str() of a torch dtype costs more than a call's other checks)


def _name(x) -> str:
    try:
        return _names[x.dtype]
    except KeyError:
        return _names.setdefault(x.dtype, str(x.dtype))


def _dense(x, what: str):
    if not x.is_contiguous():
        _refuse(f"{what} must be contiguous")


class Q8Cache:
    """One layer of a cache: codes [slots, kv_heads, cap, head_dim] (int8 or
    float8_e4m3fn), scales [slots, kv_heads, cap / 16] (float32) and the open
    blocks' tokens, tail [slots, kv_heads, 16, head_dim] (float32, bfloat16 or
    float16), for K and V. The arrays are the caller's and are kept alive."""

    __slots__ = ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "slots", "kv_heads", "cap",
                 "head_dim", "device", "dtype", "_c", "_ref")

    def __init__(self, k_codes, v_codes, k_scales, v_scales, k_tail, v_tail):
        if len(k_codes.shape) != 4:
            _refuse("codes are [slots, kv_heads, cap, head_dim]")
        s, h, cap, hd = (int(x) for x in k_codes.shape)
        kind, dtype = _KINDS.get(_name(k_codes)), _DTYPES.get(_name(k_tail))
        if kind is None:
            _refuse(f"codes are int8 or float8_e4m3fn, got {_name(k_codes)}")
        if dtype is None:
            _refuse(f"tails are float32, bfloat16 or float16, got {_name(k_tail)}")
        if cap % BLOCK:
            _refuse("cap must be a multiple of 16")
        dev = k_codes.get_device() if k_codes.is_cuda else -1
        for x, shape, name, what in ((k_codes, (s, h, cap, hd), _name(k_codes), "k_codes"),
                                     (v_codes, (s, h, cap, hd), _name(k_codes), "v_codes"),
                                     (k_scales, (s, h, cap // BLOCK), "torch.float32", "k_scales"),
                                     (v_scales, (s, h, cap // BLOCK), "torch.float32", "v_scales"),
                                     (k_tail, (s, h, BLOCK, hd), _name(k_tail), "k_tail"),
                                     (v_tail, (s, h, BLOCK, hd), _name(k_tail), "v_tail")):
            if tuple(x.shape) != shape or _name(x) != name:
                _refuse(f"{what} must be {name} {shape}, got {_name(x)} {tuple(x.shape)}")
            _dense(x, what)
            if not x.is_cuda or x.get_device() != dev:
                _refuse(f"{what} must be on the cache's CUDA device")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.k_tail, self.v_tail = k_tail, v_tail
        self.slots, self.kv_heads, self.cap, self.head_dim = s, h, cap, hd
        self.device, self.dtype = dev, k_tail.dtype
        self._c = _lib.Q8CacheC(dev, kind, dtype, s, h, cap, hd, k_codes.data_ptr(), v_codes.data_ptr(),
                                k_scales.data_ptr(), v_scales.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr())
        self._ref = ctypes.addressof(self._c)


class Q8LayerView(_lib.Q8CacheC):
    """One layer of a QuantKvCache (QuantKvCache.view), taken by q8_append,
    q8_read and q8_attend like a Q8Cache; it keeps its QuantKvCache alive."""

    owner = None
    _cache = None


def _cache_of(view) -> Q8Cache:
    """The Q8Cache that a defer_q8_cache structure describes."""
    if not isinstance(view, _lib.Q8CacheC):
        _refuse(f"the cache must be a Q8Cache or a layer's view, got {type(view).__name__}")
    c = getattr(view, "_cache", None)
    if c is None:
        t = sys.modules.get("torch")
        if t is None:
            _refuse("a layer's view needs torch arrays beside it")
        c = Q8Cache.__new__(Q8Cache)
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail"):
            setattr(c, name, None)
        c.slots, c.kv_heads, c.cap, c.head_dim, c.device = view.slots, view.kv_heads, view.cap, view.head_dim, view.device
        c.dtype = (t.float32, t.bfloat16, t.float16)[view.dtype]
        c._c, c._ref = None, ctypes.addressof(view)
        view._cache = c
    return c


def _ints(device: int, x, n: int, what: str) -> int:
    """Device pointer of an int32 array of n entries (None: NULL)."""
    if x is None:
        return 0
    if _names.get(x.dtype) != "torch.int32" or x.numel() != n or x.get_device() != device or not x.is_contiguous():
        if _name(x) != "torch.int32" or x.numel() != n or not x.is_contiguous():
            _refuse(f"{what} must be {n} contiguous int32")
        if x.get_device() != device:
            _refuse(f"{what} must be on the cache's device")
    return x.data_ptr()


def _batch(device: int, n: int, tokens: int, max_q: int, q_start, slots, status) -> bytes:
    _count(max_q, "max_q")
    return _BATCH.pack(n, tokens, max_q, _ints(device, q_start, n + 1, "q_start"), _ints(device, slots, n, "slots"),
                       0 if status is None else _ints(device, status, 1, "status"))


def _count(x: int, what: str):
    if not 0 <= x <= 0xFFFFFFFF:
        _refuse(f"{what} must be 0 to 2^32 - 1, got {x}")


def _rows(cache: Q8Cache, x, heads: int, what: str):
    """(pointer, row stride, head stride) of [tokens, heads, head_dim]."""
    shape = x.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != cache.head_dim or x.dtype != cache.dtype:
        _refuse(f"{what} must be {cache.dtype} [tokens, {heads}, {cache.head_dim}], got {x.dtype} {tuple(shape)}")
    if x.get_device() != cache.device:
        _refuse(f"{what} must be on the cache's device")
    st = x.stride()
    if st[2] != 1:
        _refuse(f"the head_dim elements of {what} must be contiguous")
    return x.data_ptr(), st[0], st[1]


def q8_append(cache: Q8Cache, k, v, pos, *, q_start=None, slots=None, max_q: int = 0, status=None,
              stream: Optional[int] = None) -> None:
    """Writes rows k, v [tokens, kv_heads, head_dim] at positions pos[i],
    pos[i] + 1, ... of each sequence i (defer_q8_append). pos, q_start, slots
    and status are int32 device arrays."""
    if not isinstance(cache, Q8Cache):
        cache = _cache_of(cache)
    dev, n = cache.device, pos.numel()
    kp, kt, kh = _rows(cache, k, cache.kv_heads, "k")
    vp, vt, vh = _rows(cache, v, cache.kv_heads, "v")
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        _refuse("k and v must have the same rows")
    rc = _lib.load().defer_q8_append(cache._ref, _batch(dev, n, tokens, max_q, q_start, slots, status),
                                     _ints(dev, pos, n, "pos"), kp, kt, kh, vp, vt, vh,
                                     _stream_of(dev) if stream is None else stream)
    if rc:
        _check(rc)


def q8_read(cache: Q8Cache, k_out, v_out, lens, *, start=None, slots=None, status=None,
            stream: Optional[int] = None) -> None:
    """Positions start[i] .. lens[i] - 1 of each sequence into k_out and v_out
    [n, kv_heads, rows, head_dim] (any strides of the first three); rows
    behind the last position are left as they were (defer_q8_read)."""
    if not isinstance(cache, Q8Cache):
        cache = _cache_of(cache)
    dev, n, shape = cache.device, lens.numel(), k_out.shape
    if len(shape) != 4 or shape[0] != n or shape[1] != cache.kv_heads or shape[3] != cache.head_dim:
        _refuse(f"k_out must be [{n}, {cache.kv_heads}, rows, {cache.head_dim}], got {tuple(shape)}")
    if v_out.shape != shape:
        _refuse("k_out and v_out must have the same shape")
    ks, vs = k_out.stride(), v_out.stride()
    for x, st, what in ((k_out, ks, "k_out"), (v_out, vs, "v_out")):
        if x.dtype != cache.dtype or x.get_device() != dev:
            _refuse(f"{what} must be {cache.dtype} on the cache's device")
        if st[3] != 1:
            _refuse(f"the head_dim elements of {what} must be contiguous")
    rc = _lib.load().defer_q8_read(cache._ref, n, _ints(dev, lens, n, "lens"), _ints(dev, start, n, "start"),
                                   _ints(dev, slots, n, "slots"), 0 if status is None else _ints(dev, status, 1, "status"),
                                   shape[2], k_out.data_ptr(), _STRIDES.pack(*ks[:3]), v_out.data_ptr(),
                                   _STRIDES.pack(*vs[:3]), _stream_of(dev) if stream is None else stream)
    if rc:
        _check(rc)


def q8_attend(cache: Q8Cache, q, out, lens, *, q_start=None, slots=None, max_q: int = 0, max_len: int = 0,
              masked=None, causal: bool = True, scale: Optional[float] = None, status=None, workspace=None,
              stream: Optional[int] = None):
    """Attention of q [tokens, heads, head_dim] over the cache into out (the
    same shape), which is returned (defer_q8_attend). lens[i] counts the
    positions of sequence i, the call's own rows among them; masked [n, cap or
    more] (uint8 or bool) hides positions; scale defaults to
    head_dim ** -0.5. Long sequences need a workspace (a contiguous device
    array of workspace_bytes() bytes or more, used while the call runs): by
    default it is taken from torch's allocator on the call's stream."""
    if not isinstance(cache, Q8Cache):
        cache = _cache_of(cache)
    dev, n = cache.device, lens.numel()
    heads = q.shape[1] if len(q.shape) == 3 else 0
    qp, qt, qh = _rows(cache, q, heads, "q")
    op, ot, oh = _rows(cache, out, heads, "out")
    tokens = q.shape[0]
    if out.shape[0] != tokens:
        _refuse("q and out must have the same rows")
    mp, ms = None, 0
    if masked is not None:
        if len(masked.shape) != 2 or masked.shape[0] != n or masked.shape[1] < cache.cap or _name(masked) not in _BYTES:
            _refuse(f"masked must be uint8 or bool [{n}, at least {cache.cap}]")
        if masked.stride(1) != 1 or masked.get_device() != dev:
            _refuse("masked must be on the cache's device with contiguous rows")
        mp, ms = masked.data_ptr(), masked.stride(0) if n > 1 else 0
    b = _batch(dev, n, tokens, max_q, q_start, slots, status)
    _count(max_len, "max_len")
    if stream is None:
        stream = _stream_of(dev)
    wp, wn = None, 0
    if workspace is not None:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            _refuse("the workspace must be contiguous on the cache's device")
        wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    elif (max_len or cache.cap) >= _LONG:
        wn = _workspace_bytes(cache, b, max_len, heads)
        if wn:
            workspace = _scratch(dev, wn, stream)  # freed in the stream's order
            wp = workspace.data_ptr()
    rc = _lib.load().defer_q8_attend(cache._ref, b, _ints(dev, lens, n, "lens"), max_len, heads, qp, qt, qh, op, ot,
                                     oh, mp, ms, 1 if causal else 0,
                                     cache.head_dim ** -0.5 if scale is None else scale, wp, wn, stream)
    if rc:
        _check(rc)
    return out


def stall_next_attend(role: int, wait_us: int = 1000) -> None:
    """Fault drill: this thread's next q8_attend of many 16-bit rows withholds
    one role's arrivals with its bounded waits cut to wait_us
    (defer_debug_q8_stall)."""
    rc = _lib.load().defer_debug_q8_stall(role, wait_us)
    if rc:
        _check(rc)


_LONG = 9000  # shorter sequences need no workspace, whatever the head size


def _workspace_bytes(cache: Q8Cache, batch: bytes, max_len: int, heads: int) -> int:
    n = ctypes.c_size_t(0)
    rc = _lib.load().defer_q8_attend_workspace(cache._ref, batch, max_len, heads, ctypes.byref(n))
    if rc:
        _check(rc)
    return n.value


def workspace_bytes(cache: Q8Cache, tokens: int, heads: int, max_len: int = 0, *, n: Optional[int] = None) -> int:
    """Bytes of workspace with which q8_attend of `tokens` rows of `heads`
    heads and this max_len runs, however the rows belong to sequences; with
    `n`, of a call without q_start whose n sequences have tokens / n rows each
    (defer_q8_attend_workspace; many rows a sequence need none)."""
    if not isinstance(cache, Q8Cache):
        cache = _cache_of(cache)
    for x, what in ((tokens, "tokens"), (heads, "heads"), (max_len, "max_len"), (n or 0, "n")):
        _count(x, what)
    # the host only asks whether there is a q_start: with one, sequences may have any number of rows
    b = _BATCH.pack(1, tokens, 0, 1, 0, 0) if n is None else _BATCH.pack(n, tokens, 0, 0, 0, 0)
    return _workspace_bytes(cache, b, max_len, heads)


def _scratch(device: int, nbytes: int, stream: int):
    t = sys.modules.get("torch")
    if t is None:
        _refuse("a sequence this long needs the workspace argument")
    if stream == t.cuda.current_stream(device).cuda_stream:
        return t.empty(nbytes, dtype=t.uint8, device=f"cuda:{device}")
    # 0 is the default stream; an ExternalStream of 0 would be one of torch's own
    s = t.cuda.ExternalStream(stream, device=device) if stream else t.cuda.default_stream(device)
    with t.cuda.stream(s):
        return t.empty(nbytes, dtype=t.uint8, device=f"cuda:{device}")
