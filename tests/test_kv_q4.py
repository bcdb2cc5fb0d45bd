"""The 4-bit KV cache and the key window of layers and models, on the CPU: the
oracle's Q4_0 cache (RefLayer(kv="q4")) against the host quantiser's blocks, its
window against full attention and against a copy of the visible keys, and the
layer config's mapping."""
import numpy as np
import pytest

import oracle
from flock_b200 import _abi, synth
from flock_b200 import lib as flib
from flock_b200.layer import QWEN3_06B

CFG = dict(hidden=64, n_heads=2, n_kv_heads=1, head_dim=128, ffn=64)


@pytest.fixture(scope="module")
def weights():
    rng = np.random.default_rng(3)
    rows = {"attn_q.weight": (256, 64), "attn_k.weight": (128, 64), "attn_v.weight": (128, 64),
            "attn_output.weight": (64, 256), "ffn_gate.weight": (64, 64),
            "ffn_up.weight": (64, 64), "ffn_down.weight": (64, 64)}
    out = {n: oracle.quant_matrix_q8(rng.standard_normal(r * c).astype(np.float32), r, c)
           for n, (r, c) in rows.items()}
    for n, size in (("attn_norm.weight", 64), ("ffn_norm.weight", 64),
                    ("attn_q_norm.weight", 128), ("attn_k_norm.weight", 128)):
        out[n] = 1 + 0.1 * rng.standard_normal(size).astype(np.float32)
    return out


def q4(x):
    packed = flib.quant_matrix_q4(x.reshape(-1, 32), x.size // 32, 32).reshape(-1, 18)
    d = packed[:, :2].copy().view(np.float16).astype(np.float64)
    codes = np.concatenate([packed[:, 2:] & 15, packed[:, 2:] >> 4], 1).astype(np.float64) - 8
    return (codes * d).astype(np.float32).reshape(x.shape)


@pytest.mark.parametrize("scale", [1e-6, 1.0, 300.0])
def test_oracle_cache_keeps_q4_blocks(weights, scale):
    x = np.random.default_rng(4).standard_normal((5, 128)).astype(np.float32) * np.float32(scale)
    x[2, 32:64] = 0
    ref = oracle.RefLayer(weights, CFG, 8, kv="q4")
    ref.fill_cache(x, -x)
    k, v = ref.cache()
    assert np.array_equal(k, q4(x).ravel()) and np.array_equal(v, q4(-x).ravel())
    again = oracle.RefLayer(weights, CFG, 8, kv="q4")   # stored values store as themselves
    again.fill_cache(k, v)
    assert np.array_equal(again.cache()[0], k) and np.array_equal(again.cache()[1], v)


def test_oracle_window_that_holds_everything(weights):
    x = np.random.default_rng(5).standard_normal((9, 64)).astype(np.float32)
    a, b = oracle.RefLayer(weights, CFG, 16), oracle.RefLayer(weights, CFG, 16)
    b.set_window(9)
    # Attention is rounded once here and per operation there: a relative 128 * 2^-24 at most.
    # The outputs reach 1e3, where one f32 step is 6e-5: the bound is relative to the largest,
    # 1e-5 of it as for the layers' fast attention (typical: 128^0.5 * 2^-24 = 7e-7).
    want = a.forward(x, 9)
    assert np.abs(want - b.forward(x, 9)).max() < 1e-5 * np.abs(want).max()
    assert np.abs(a.forward(x[0], 1) - b.forward(x[0], 1)).max() > 1e-6   # ten keys, nine seen


def test_oracle_window_sees_sinks_and_newest(weights):
    """A decode step in a window equals one over a cache of the visible keys; the
    hidden ones do not count, whatever they hold.  (Rotations are stored with the
    keys, so the copy starts at the same position by filling hidden rows.)"""
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((20, 128)).astype(np.float32) for _ in range(2))
    x = rng.standard_normal(64).astype(np.float32)
    a, b = oracle.RefLayer(weights, CFG, 32), oracle.RefLayer(weights, CFG, 32)
    for L in (a, b):
        L.set_window(6, 2)
    a.fill_cache(k, v)
    k2, v2 = k.copy(), v.copy()
    k2[2:15], v2[2:15] = 50.0, np.nan     # the step is key 20: it sees 0, 1 and 15 .. 20
    b.fill_cache(k2, v2)
    assert np.array_equal(a.forward(x, 1), b.forward(x, 1))


def test_config_maps_q4():
    c = QWEN3_06B.with_(attention="fast", prefill="tensor", kv="q4").to_c()
    assert c.kv_dtype == _abi.FLOCK_KV_Q4 == 3


def test_set_window_refuses_null():
    lib = _abi.lib()
    assert lib.flock_layer_set_window(None, 4, 0) < 0
    assert lib.flock_model_set_window(None, 4, 0) < 0
