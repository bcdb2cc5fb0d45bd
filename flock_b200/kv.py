"""KV caches in device memory and the attention that reads them.

For callers that keep queries, keys and logits on the GPU themselves (a
serving loop, a draft model beside the target).  Arrays are device arrays: a
torch CUDA tensor, or anything with ``__cuda_array_interface__``.

    cache = KVCache(dev, "q4", n_kv_heads=8, capacity=32768)
    cache.append(k, v, pos)                       # f32 rows into the cache
    cache.attention(q, pos, out, window=4096, sinks=4)

``stream`` is a cudaStream_t as an integer (torch:
``torch.cuda.current_stream().cuda_stream``); 0 is the default stream.  Calls
enqueue work and return: order them against other streams yourself.
"""
from __future__ import annotations

import ctypes
import math

from . import _abi
from .lib import Device

KV_DTYPES = {"f32": _abi.FLOCK_KV_F32, "bf16": _abi.FLOCK_KV_BF16, "fp8": _abi.FLOCK_KV_FP8,
             "q4": _abi.FLOCK_KV_Q4}
HEAD_DIM = 128
# ctypes keeps an integer's low bits, so what the C types cannot hold is brought
# to the nearest number that they can: no cache is as long as either.
_INT_MAX = 2 ** 31 - 1   # a window past it sees every key
_POS_MAX = 2 ** 63 - 1   # outside of every cache, as is -1
WORKSPACE_BYTES = _abi.FLOCK_WORKSPACE_BYTES

# __cuda_array_interface__ type strings and torch dtype names of an element
_TYPES = {"f32": ("<f4", "float32"), "bf16": ("<u2", "bfloat16"), "fp8": ("|u1", "float8_e4m3fn"),
          "u8": ("|u1", "uint8"), "f16": ("<f2", "float16"), "i32": ("<i4", "int32")}
_torch_types: dict = {}  # torch dtype -> element name, filled when a tensor comes by


def _position(pos: int) -> int:
    return -1 if pos < 0 else pos if pos <= _POS_MAX else _POS_MAX


def _window(n: int) -> int:
    """A window or a number of sinks; negative ones stay so, to be refused."""
    return -1 if n < 0 else n if n <= _INT_MAX else _INT_MAX


def _torch_type(t) -> str | None:
    if not _torch_types:
        import torch  # a torch tensor is here, so torch is loaded
        _torch_types.update({getattr(torch, n): e for e, (_, n) in _TYPES.items()})
    return _torch_types.get(t)


def _array(a, dtype: str, ordinal: int, what: str):
    """(device address, shape, strides in elements or None when dense)."""
    try:
        t, p = a.dtype, a.data_ptr()
    except AttributeError:
        return _interface(a, dtype, ordinal, what)
    if (_torch_types.get(t) or _torch_type(t)) != dtype:
        raise ValueError(f"{what} is {t}, want torch.{_TYPES[dtype][1]}")
    if a.get_device() != ordinal:  # -1 on the host
        raise ValueError(f"{what} is on {a.device}, the cache's device is cuda:{ordinal}")
    return p, a.shape, None if a.is_contiguous() else a.stride()


def _interface(a, dtype: str, ordinal: int, what: str):
    i = getattr(a, "__cuda_array_interface__", None)
    if i is None:
        raise ValueError(f"{what} is a {type(a).__name__}, not a device array")
    if i["typestr"] != _TYPES[dtype][0]:
        raise ValueError(f"{what} has type {i['typestr']}, want {_TYPES[dtype][0]}")
    at, shape, strides = i["data"][0], tuple(i["shape"]), i.get("strides")
    on = _abi.lib().flock_pointer_device(at or None)
    if on >= 0 and on != ordinal:
        raise ValueError(f"{what} is on cuda:{on}, the cache's device is cuda:{ordinal}")
    if strides is None:
        return at, shape, None
    size = int(i["typestr"][2:])
    if any(n > 1 and s % size for n, s in zip(shape, strides)):
        raise ValueError(f"{what} has strides of {tuple(strides)} bytes, not of whole elements")
    strides = tuple(s // size for s in strides)
    dense = all(n == 1 or s == math.prod(shape[d + 1:]) for d, (n, s) in enumerate(zip(shape, strides)))
    return at, shape, None if dense or 0 in shape else strides


def _stream_of(a) -> int:
    """The stream that a device array is written on, as far as it says: torch's
    current one, or the interface's (none named: 0, the default stream)."""
    if hasattr(a, "data_ptr"):
        import torch
        return torch.cuda.current_stream(a.device).cuda_stream if a.is_cuda else 0
    return getattr(a, "__cuda_array_interface__", {}).get("stream") or 0


def _dense(a, dtype: str, ordinal: int, what: str, shape: tuple) -> int:
    p, got, strides = _array(a, dtype, ordinal, what)
    if strides is not None or tuple(got) != shape:
        raise ValueError(f"{what} is {tuple(got)}{'' if strides is None else ' with strides'}, "
                         f"want a dense {shape}")
    return p


def _rows(a, ordinal: int, what: str, heads: int | None) -> tuple:
    """An f32 [n][heads][128] whose rows may be further apart: (address, n,
    heads, row stride in floats)."""
    p, shape, strides = _array(a, "f32", ordinal, what)
    if len(shape) != 3 or shape[2] != HEAD_DIM or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} is {tuple(shape)}, want [n][{heads or 'heads'}][{HEAD_DIM}]")
    if strides is None:
        return p, shape[0], shape[1], 0
    if (strides[2] != 1 or (shape[1] > 1 and strides[1] != HEAD_DIM) or
            (shape[0] > 1 and strides[0] < shape[1] * HEAD_DIM)):
        raise ValueError(f"{what} has strides {tuple(strides)}: each row's heads must be dense")
    return p, shape[0], shape[1], strides[0] if shape[0] > 1 else 0


class KVCache:
    """flock_kv: a cache of ``capacity`` keys.  ``k`` and ``v`` (and, for "q4",
    ``k_scales`` and ``v_scales``) are the caller's planes, kept alive here;
    without them the cache allocates its own, zero-filled.

    f32, bf16 and fp8 planes are [capacity][n_kv_heads][128]; "q4" planes are
    uint8 [n_kv_heads][capacity][64] with f16 scales [n_kv_heads][capacity][4]
    (include/flock_cuda.h has the bytes' order), capacity a multiple of 16.
    ``workspace``: WORKSPACE_BYTES of zero-filled uint8 that only this cache's
    attention uses; attention calls of one KVCache must not overlap on the GPU.
    """

    def __init__(self, dev: Device, dtype: str, n_kv_heads: int, capacity: int, k=None, v=None,
                 k_scales=None, v_scales=None, workspace=None, head_dim: int = HEAD_DIM):
        self.handle = None
        if dtype not in KV_DTYPES:
            raise ValueError(f"kv dtype {dtype!r} is not one of {sorted(KV_DTYPES)}")
        self.dev, self.dtype, self.n_kv_heads, self.capacity = dev, dtype, n_kv_heads, capacity
        self._keep = (dev, k, v, k_scales, v_scales, workspace)
        o = dev.ordinal
        if dtype == "q4":
            row, srow = (n_kv_heads, capacity, 64), (n_kv_heads, capacity, 4)
            planes = [a if a is None else _dense(a, "u8", o, w, row)
                      for a, w in ((k, "k"), (v, "v"))]
            planes += [a if a is None else _dense(a, "f16", o, w, srow)
                       for a, w in ((k_scales, "k_scales"), (v_scales, "v_scales"))]
        else:
            if k_scales is not None or v_scales is not None:
                raise ValueError(f"a {dtype} cache has no scales")
            row = (capacity, n_kv_heads, HEAD_DIM)
            planes = [a if a is None else _dense(a, dtype, o, w, row)
                      for a, w in ((k, "k"), (v, "v"))] + [None, None]
        ws = None if workspace is None else _workspace(workspace, o)
        h = ctypes.c_void_p()
        _abi.call("flock_kv_create", dev.handle, KV_DTYPES[dtype], n_kv_heads, head_dim, capacity,
                  *planes, ws, ctypes.byref(h))
        self.handle = h
        # the entry points, looked up once
        lib = _abi.lib()
        self._append, self._read = lib.flock_kv_append, lib.flock_kv_read
        self._attention = lib.flock_kv_attention

    def free(self) -> None:
        if self.handle:
            _abi.lib().flock_kv_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def append(self, k, v, pos: int, stream: int = 0) -> None:
        """Round f32 rows k and v [n][n_kv_heads][128] into positions pos ..
        pos + n - 1.  Rows may be further apart than dense, k and v alike."""
        kp, n, _, ks = _rows(k, self.dev.ordinal, "k", self.n_kv_heads)
        vp, nv, _, vs = _rows(v, self.dev.ordinal, "v", self.n_kv_heads)
        if n != nv or ks != vs:
            raise ValueError(f"k has {n} rows at stride {ks}, v {nv} at {vs}")
        rc = self._append(self.handle, kp, vp, ks, _position(pos), n, stream or None)
        if rc:
            _abi.check(rc)

    def read(self, pos: int, n: int, k, v, stream: int = 0) -> None:
        """The cached rows pos .. pos + n - 1 into f32 k and v [n][n_kv_heads][128]."""
        shape = (n, self.n_kv_heads, HEAD_DIM)
        rc = self._read(self.handle, _position(pos), n, _dense(k, "f32", self.dev.ordinal, "k", shape),
                        _dense(v, "f32", self.dev.ordinal, "v", shape), stream or None)
        if rc:
            _abi.check(rc)

    def attention(self, q, pos: int, out, window: int = 0, sinks: int = 0,
                  stream: int = 0) -> None:
        """Causal attention of q [n][n_heads][128] f32 at positions pos .. pos +
        n - 1 over the cache's keys up to each, into out of the same shape.
        ``window`` > 0 limits a query at p to keys j > p - window and the first
        ``sinks`` keys."""
        qp, n, heads, qs = _rows(q, self.dev.ordinal, "q", None)
        op, no, _, os_ = _rows(out, self.dev.ordinal, "out", heads)
        if no != n:
            raise ValueError(f"out has {no} rows, q {n}")
        rc = self._attention(self.handle, qp, qs, heads, n, _position(pos), _window(window),
                             _window(sinks), op, os_, stream or None)
        if rc:
            _abi.check(rc)


class DraftVerifier:
    """flock_verify_draft over a vocabulary: drafted tokens checked against the
    target's logits with given uniform numbers.  ``workspace``: WORKSPACE_BYTES
    of device uint8, 16-byte aligned, that no overlapping call uses."""

    def __init__(self, dev: Device, vocab: int, workspace):
        self.dev, self.vocab = dev, vocab
        self._keep = workspace
        self._ws = _workspace(workspace, dev.ordinal)
        if self._ws & 15:
            raise ValueError("the workspace is not 16-byte aligned")
        self._verify = _abi.lib().flock_verify_draft

    def _logits(self, a, what: str, n: int, rows: int) -> tuple:
        p, shape, st = _array(a, "f32", self.dev.ordinal, what)
        if tuple(shape) != (n, rows, self.vocab):
            raise ValueError(f"{what} is {tuple(shape)}, want {(n, rows, self.vocab)}")
        if st is None:
            return p, 0
        step = st[1] if rows > 1 else st[0]
        if st[2] != 1 or (n > 1 and st[0] != rows * step) or step < self.vocab:
            raise ValueError(f"{what} has strides {tuple(st)}: rows must be evenly spaced")
        return p, step

    def verify(self, target, draft, ids, u, tokens, accepted, lens=None,
               temperature: float = 1.0, stream: int = 0) -> None:
        """target [n][d + 1][vocab] f32, draft [n][d][vocab] f32 or None, ids
        [n][d] i32, u [n][d + 1] f32 in [0, 1), lens [n] i32 or None; into
        tokens [n][d + 1] and accepted [n], i32.  include/flock_cuda.h
        flock_verify_draft has the rule."""
        o = self.dev.ordinal
        ip, (n, d), st = _array(ids, "i32", o, "ids")
        if st is not None:
            raise ValueError("ids must be dense")
        tp, ts = self._logits(target, "target", n, d + 1)
        dp, ds = (None, 0) if draft is None else self._logits(draft, "draft", n, d)
        rc = self._verify(self.dev.handle, tp, ts, dp, ds, ip, _dense(u, "f32", o, "u", (n, d + 1)),
                          None if lens is None else _dense(lens, "i32", o, "lens", (n,)), n, d,
                          self.vocab, temperature, _dense(tokens, "i32", o, "tokens", (n, d + 1)),
                          _dense(accepted, "i32", o, "accepted", (n,)), self._ws, stream or None)
        if rc:
            _abi.check(rc)


def _workspace(a, ordinal: int) -> int:
    p, shape, strides = _array(a, "u8", ordinal, "workspace")
    if strides is not None or math.prod(shape) < WORKSPACE_BYTES:
        raise ValueError(f"workspace has {math.prod(shape)} bytes, want {WORKSPACE_BYTES} dense")
    return p
