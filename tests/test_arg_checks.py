"""The entry points' argument checks without a GPU: csrc/arg_checks.h compiled by
itself."""
import ctypes
import os
import subprocess

import pytest

from flock_b200 import _abi, kv

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
