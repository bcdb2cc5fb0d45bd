"""flock_kv_*, flock_verify_draft and flock_model_step_draft without a GPU: what
the entry points refuse before they touch a device, with the error text set, and
what the Python classes refuse before they call them."""
import ctypes

import numpy as np
import pytest

from flock_b200 import _abi, kv

E_ARG = -1


class FakeDevice:
    ordinal = 0
    handle = None


class OnDevice:
    """What a CUDA array shows of itself; nothing reads the address here."""

    def __init__(self, shape, typestr, strides=None):
        self.__cuda_array_interface__ = dict(shape=shape, typestr=typestr, strides=strides,
                                             data=(4096, False), version=3)


def _refused(name, *args, word):
    lib = _abi.lib()
    assert getattr(lib, name)(*args) == E_ARG
    assert word in lib.flock_last_error().decode()


def test_null_arguments():
    h = ctypes.c_void_p()
    n = ctypes.c_int()
    _refused("flock_kv_create", None, 3, 8, 128, 64, None, None, None, None, None,
             ctypes.byref(h), word="kv_create")
    _refused("flock_kv_append", None, None, None, 0, 0, 1, None, word="kv_append")
    _refused("flock_kv_read", None, 0, 1, None, None, None, word="kv_read")
    _refused("flock_kv_attention", None, None, 0, 16, 1, 0, 0, 0, None, 0, None,
             word="kv_attention")
    _refused("flock_verify_draft", None, None, 0, None, 0, None, None, None, 1, 1, 32, 1.0, None,
             None, None, None, word="verify_draft")
    _refused("flock_model_step_draft", None, None, 1, None, None, 0.0, None, ctypes.byref(n),
             word="step_draft")
    assert _abi.lib().flock_kv_free(None) == 0


def test_cache_names_its_types():
    with pytest.raises(ValueError, match="q4"):
        kv.KVCache(FakeDevice(), "int4", 8, 64)


@pytest.mark.parametrize("bad", [np.zeros(kv.WORKSPACE_BYTES, np.uint8), [1, 2],
                                 OnDevice((kv.WORKSPACE_BYTES - 16,), "|u1"),
                                 OnDevice((kv.WORKSPACE_BYTES // 4,), "<f4"),
                                 OnDevice((kv.WORKSPACE_BYTES,), "|u1", (2,))])
def test_workspace_is_checked(bad):
    with pytest.raises(ValueError, match="workspace"):
        kv.DraftVerifier(FakeDevice(), 32000, bad)


def test_verifier_checks_shapes():
    v = kv.DraftVerifier(FakeDevice(), 100, OnDevice((kv.WORKSPACE_BYTES,), "|u1"))
    good = dict(target=OnDevice((2, 4, 100), "<f4"), draft=OnDevice((2, 3, 100), "<f4"),
                ids=OnDevice((2, 3), "<i4"), u=OnDevice((2, 4), "<f4"),
                tokens=OnDevice((2, 4), "<i4"), accepted=OnDevice((2,), "<i4"))
    for name, bad in [("target", OnDevice((2, 3, 100), "<f4")),
                      ("target", OnDevice((2, 4, 100), "<f2")),
                      ("target", OnDevice((2, 4, 100), "<f4", (1600, 400, 8))),
                      ("draft", OnDevice((2, 3, 99), "<f4")), ("u", OnDevice((2, 3), "<f4")),
                      ("ids", OnDevice((2, 3), "<i4", (40, 4))), ("tokens", OnDevice((2, 3), "<i4")),
                      ("accepted", OnDevice((3,), "<i4")), ("lens", OnDevice((1,), "<i4"))]:
        with pytest.raises(ValueError, match=name):
            v.verify(**{**good, name: bad})
