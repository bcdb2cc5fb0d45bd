"""The entry points' argument checks without a GPU: csrc/arg_checks.h compiled by
itself, and the integers that kv.py and the model classes hand on."""
import ctypes
import os
import subprocess
import types

import pytest

from flock_b200 import _abi, kv
from flock_b200.layer import Layer
from flock_b200.model import Model

CSRC = os.path.join(os.path.dirname(_abi.__file__), "csrc")
I64_MAX, I64_MIN = 2 ** 63 - 1, -2 ** 63


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    """The header's functions with C names, at the optimisation they ship with."""
    d = tmp_path_factory.mktemp("arg_checks")
    src, so = d / "checks.cc", d / "checks.so"
    src.write_text('#include "arg_checks.h"\nextern "C" int range_inside(int64_t p, int64_t n, '
                   'int64_t c) { return flock::range_inside(p, n, c); }\n')
    subprocess.run(["g++", "-O3", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.range_inside.argtypes = [ctypes.c_int64] * 3
    return lib


@pytest.mark.parametrize("capacity", [1, 32, 2 ** 30])
def test_positions_inside_a_cache(checks, capacity):
    """Against the same question in unbounded integers, at every border."""
    some = {0, 1, 2, 31, 32, 33, capacity - 1, capacity, capacity + 1, 2 ** 31 - 1, 2 ** 31,
            I64_MAX - 1, I64_MAX}
    for pos in some | {-x for x in some} | {I64_MIN, I64_MAX - capacity}:
        for n in (-1, 0, 1, 2, 32, capacity, 2 ** 31 - 1):
            want = pos >= 0 and n >= 0 and pos + n <= capacity
            assert checks.range_inside(pos, n, capacity) == want, (pos, n, capacity)


class OnDevice:
    """What a CUDA array shows of itself; nothing reads the address here."""

    def __init__(self, *shape):
        self.__cuda_array_interface__ = dict(shape=shape, typestr="<f4", strides=None,
                                             data=(4096, False), version=3)


def _cache(name):
    """A KVCache whose `name` entry point records what reaches the C call."""
    seen = []
    c = object.__new__(kv.KVCache)
    c.handle, c.dev, c.n_kv_heads = None, types.SimpleNamespace(ordinal=0), 2
    proto = ctypes.CFUNCTYPE(ctypes.c_int, *_abi.SIGNATURES[f"flock_kv_{name}"])
    c._entry = proto(lambda *a: seen.append(a) or 0)
    setattr(c, f"_{name}", c._entry)
    return c, seen


@pytest.mark.parametrize("pos", [2 ** 63, 2 ** 64, 2 ** 64 + 3, -2 ** 63 - 1, -2 ** 64])
def test_a_position_past_64_bits_is_not_another_one(checks, pos):
    """ctypes keeps the low 64 bits of an integer: 2^64 + 3 must not become 3."""
    x = OnDevice(1, 2, 128)
    for name, at, call in [("append", 4, lambda c: c.append(x, x, pos)),
                           ("read", 1, lambda c: c.read(pos, 1, x, x)),
                           ("attention", 5, lambda c: c.attention(x, pos, x))]:
        c, seen = _cache(name)
        call(c)
        assert not checks.range_inside(seen[0][at], 1, 2 ** 30), name


@pytest.mark.parametrize("window,sinks", [(-2 ** 32, 0), (5, -2 ** 32), (-2 ** 31 - 1, 1)])
def test_a_negative_window_stays_negative(monkeypatch, window, sinks):
    x = OnDevice(1, 2, 128)
    c, seen = _cache("attention")
    c.attention(x, 0, x, window=window, sinks=sinks)
    assert seen[0][6] < 0 or seen[0][7] < 0
    for cls, name in ((Layer, "flock_layer_set_window"), (Model, "flock_model_set_window")):
        args = []
        monkeypatch.setattr(_abi, "call", lambda fn, handle, *a: args.append((fn, a)))
        o = object.__new__(cls)
        o.handle = None
        o.set_window(window, sinks)
        fn, (w, s) = args[0]
        assert fn == name and -2 ** 31 <= min(w, s) < 0 and max(w, s) < 2 ** 31


def test_windows_past_32_bits_see_every_key():
    x = OnDevice(1, 2, 128)
    c, seen = _cache("attention")
    c.attention(x, 0, x, window=2 ** 40, sinks=2 ** 33)
    assert seen[0][6] == seen[0][7] == 2 ** 31 - 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "q4"])
def test_positions_whose_end_passes_64_bits_are_refused(dtype):
    """Refused on the host: no kernel is launched."""
    import torch
    from flock_b200 import lib as flib
    cache = kv.KVCache(flib.get_device(0), dtype, 2, 32)
    x, out = (torch.zeros(2, 2, 128, device="cuda") for _ in range(2))
    for pos in (I64_MAX, I64_MAX - 1, 2 ** 62, 31, -1):
        for call in (lambda: cache.append(x, x, pos), lambda: cache.read(pos, 2, x, out),
                     lambda: cache.attention(x, pos, out)):
            with pytest.raises(_abi.FlockError, match="inside a cache") as e:
                call()
            assert e.value.code == _abi.FLOCK_E_STATE
    cache.append(x, x, 30)
    cache.attention(x, 30, out)


# ------------------------------------------------- draft verification's addresses
# target, draft, ids, u, lens, tokens, accepted, workspace: argument numbers
ADDRESSES = dict(target=1, draft=3, ids=5, u=6, lens=7, tokens=12, accepted=13, workspace=14)


def _verify(temperature, **at):
    """flock_verify_draft with made-up addresses, refused before a device is touched."""
    dev = ctypes.create_string_buffer(1024)   # no device; its first bytes say ordinal 0
    args = [ctypes.addressof(dev), 4096, 0, 4096, 0, 4096, 4096, 4096, 1, 2, 100, temperature,
            4096, 4096, 4096, None]
    for name, a in at.items():
        args[ADDRESSES[name]] = a
    lib = _abi.lib()
    return lib.flock_verify_draft(*args), lib.flock_last_error().decode()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("name,off", [("workspace", 1), ("workspace", 4), ("workspace", 8)] +
                         [(n, 2) for n in ADDRESSES if n != "workspace"])
def test_misaligned_addresses_are_refused(name, off, temperature):
    rc, text = _verify(temperature, **{name: 4096 + off})
    assert rc == _abi.FLOCK_E_ARG and "aligned" in text


class Bytes:
    def __init__(self, at):
        self.__cuda_array_interface__ = dict(shape=(kv.WORKSPACE_BYTES,), typestr="|u1",
                                             strides=None, data=(at, False), version=3)


def test_a_misaligned_workspace_is_refused():
    dev = types.SimpleNamespace(ordinal=0, handle=None)
    kv.DraftVerifier(dev, 100, Bytes(4096))
    for at in (4097, 4100, 4104):
        with pytest.raises(ValueError, match="workspace.*aligned"):
            kv.DraftVerifier(dev, 100, Bytes(at))


# ------------------------------------------------------- where an array is written
def test_the_stream_that_an_array_names():
    class On:
        def __init__(self, **kw):
            self.__cuda_array_interface__ = dict(shape=(1,), typestr="<f4", data=(4096, False),
                                                 version=3, **kw)
    assert [kv._stream_of(On()), kv._stream_of(On(stream=None)), kv._stream_of(On(stream=2)),
            kv._stream_of(On(stream=77)), kv._stream_of([1.0])] == [0, 0, 2, 77, 0]


def test_wait_stream_wants_a_model():
    assert _abi.lib().flock_model_wait_stream(None, None) == _abi.FLOCK_E_ARG
    assert "wait_stream" in _abi.lib().flock_last_error().decode()


# ------------------------------------------------------- __cuda_array_interface__
class Array:
    def __init__(self, shape, strides, typestr="<f4"):
        self.__cuda_array_interface__ = dict(shape=shape, typestr=typestr, strides=strides,
                                             data=(4096, False), version=3)


def test_an_array_of_another_device_is_refused(monkeypatch):
    a = Array((2, 2, 128), None)
    assert kv._array(a, "f32", 0, "x") == (4096, (2, 2, 128), None)
    for on in (0, 1, 5, -1):   # -1: the runtime does not know the address
        monkeypatch.setattr(_abi, "lib", lambda: types.SimpleNamespace(flock_pointer_device=lambda p: on))
        if on in (0, -1):
            assert kv._array(a, "f32", 0, "x")[0] == 4096
        else:
            with pytest.raises(ValueError, match=f"x is on cuda:{on}"):
                kv._array(a, "f32", 0, "x")


def test_dense_strides_are_dense():
    for shape, strides in [((2, 3, 128), (1536, 512, 4)), ((1, 3, 128), (99, 512, 4)),
                           ((0, 3, 128), (0, 0, 4)), ((5,), (4,))]:
        assert kv._array(Array(shape, strides), "f32", 0, "x")[2] is None
    assert kv._array(Array((2, 3, 128), (2048, 512, 4)), "f32", 0, "x")[2] == (512, 128, 1)
    assert kv._dense(Array((2, 3), (12, 4)), "f32", 0, "x", (2, 3)) == 4096


def test_strides_of_parts_of_elements_are_refused():
    with pytest.raises(ValueError, match="whole elements"):
        kv._array(Array((2, 3), (18, 6)), "f32", 0, "x")


@pytest.mark.gpu
def test_the_device_of_a_pointer():
    import torch
    f = _abi.lib().flock_pointer_device
    x = torch.zeros(4, device="cuda")
    assert f(x.data_ptr()) == 0 and f(x.data_ptr() + 4) == 0
    assert f(torch.zeros(4).data_ptr()) == -1 and f(torch.zeros(4).pin_memory().data_ptr()) == -1
    assert f(None) == -1 and f(4096) == -1
    x.add_(1)   # no error is left behind
    torch.cuda.synchronize()
