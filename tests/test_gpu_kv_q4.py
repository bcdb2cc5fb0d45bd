"""Layers and models over a 4-bit KV cache (kv="q4", FLOCK_KV_Q4) and with a key
window (set_window) on the GPU: stored rows equal to the oracle's, read back
exactly; decode steps over preloaded rows within the fast-attention bound 1e-5
absErrScaled; the tensor-core prefill within its 1e-2 bound of a 64-bit
attention over the rows that it stored; decode graphs, windows changed between
steps, and tensors that a window hides; engines that fall back; refusals."""
import numpy as np
import pytest

from flock_b200 import lib as flib
from flock_b200 import synth
from flock_b200._abi import FlockError
from flock_b200.layer import QWEN3_06B, Layer
from flock_b200.model import Model
from gpu_util import abs_err_scaled, bits, n_mismatch

pytestmark = pytest.mark.gpu

S = synth.QWEN3_06B
CFG = dict(hidden=S.hidden, n_heads=S.n_heads, n_kv_heads=S.n_kv_heads, head_dim=S.head_dim,
           ffn=S.ffn)
KVW = S.n_kv_heads * S.head_dim
FAST = QWEN3_06B.with_(attention="fast", prefill="tensor")


@pytest.fixture(scope="module")
def dev():
    d = flib.get_device(0)
    yield d
    d.close()


@pytest.fixture(scope="module")
def weights():
    return synth.layer_weights(110, 24)


def _ref(oracle, weights, kv, cap, window=(0, 0)):
    oracle.set_fma_mode(False)
    ref = oracle.RefLayer(weights, CFG, cap, kv=kv)
    ref.set_window(*window)
    return ref


def test_write_rounds_read_widens(dev, oracle, weights):
    """Capacity 21 is not whole 16-key groups; rows go in at two offsets."""
    kc = synth.normal(511, "k", 21 * KVW) * np.float32(40.0)
    vc = synth.normal(511, "v", 21 * KVW) * np.float32(1e-6)   # scales below f16's normals
    L = Layer.create(dev, weights, FAST.with_(kv="q4", max_keys=21))
    assert L.cache_buffers()[0].size == 0
    L.write_cache(kc[:0], vc[:0])
    L.write_cache(kc[:5 * KVW], vc[:5 * KVW])
    L.write_cache(kc[5 * KVW:], vc[5 * KVW:])
    ref = _ref(oracle, weights, "q4", 21)
    ref.fill_cache(kc, vc)
    for got, want in zip(L.cache_buffers(), ref.cache()):
        assert np.array_equal(got, want)   # (a zero's sign is not kept)


# decode: the preloaded rows are equal on both sides, so the fast-attention bound holds
@pytest.mark.parametrize("kv,n_cache,window", [
    ("q4", 1, (0, 0)), ("q4", 256, (0, 0)), ("q4", 5000, (0, 0)), ("q4", 5000, (300, 4)),
    ("f32", 700, (129, 0)), ("f32", 700, (1, 0)), ("bf16", 2100, (512, 17)),
    ("fp8", 2100, (2000, 1))])
def test_decode_over_preloaded_cache(dev, oracle, weights, kv, n_cache, window):
    kc = synth.normal(512, f"k{n_cache}", n_cache * KVW)
    vc = synth.normal(512, f"v{n_cache}", n_cache * KVW)
    L = Layer.create(dev, weights, FAST.with_(kv=kv, max_keys=n_cache + 8))
    L.set_window(*window)
    L.write_cache(kc, vc)
    ref = _ref(oracle, weights, kv, n_cache + 8, window)
    ref.fill_cache(kc, vc)
    for step in range(3):
        x = synth.normal(513, f"x{step}", S.hidden)
        e = abs_err_scaled(L.forward(x), ref.forward(x, 1))
        print(f"{kv}, {n_cache} keys, step {step}: absErrScaled {e:.2e}")
        assert e < 1e-5
    (k, v), (rk, rv) = L.cache_buffers(), ref.cache()
    assert L.n_keys == n_cache + 3
    old = n_cache * KVW
    assert np.array_equal(k[:old], rk[:old]) and np.array_equal(v, rv)
    assert np.count_nonzero(k[old:] != rk[old:]) <= 2


def _layer_from_rows(oracle, w, x, k, v, pos, window, sinks):
    """The layer's output for hidden rows x at pos over the given cache rows."""
    n, H, hd, nh = len(x), S.hidden, S.head_dim, S.n_heads
    packed = {m: (t["packed"] if isinstance(t, dict) else t) for m, t in w.items()}

    def mv(name, a, rows, cols):
        return oracle.matmul_q8_batched(packed[name], a, rows, cols, n)
    nh_ = oracle.rmsnorm(x.ravel(), packed["attn_norm.weight"], H, n)
    q = mv("attn_q.weight", nh_, nh * hd, H)
    q = oracle.rope(oracle.rmsnorm(q, packed["attn_q_norm.weight"], hd, n * nh), n, nh, hd, pos,
                    oracle.rope_inv_freq(hd, 1e6)).reshape(n, nh, hd).astype(np.float64)
    k = k.reshape(-1, S.n_kv_heads, hd).astype(np.float64)
    v = v.reshape(-1, S.n_kv_heads, hd).astype(np.float64)
    attn = np.zeros((n, nh, hd))
    for i in range(n):
        p = pos + i
        keys = [t for t in range(p + 1) if not window or t < sinks or t > p - window]
        for h in range(nh):
            kv = h // (nh // S.n_kv_heads)
            s = k[keys, kv] @ q[i, h] / np.sqrt(hd)
            e = np.exp(s - s.max())
            attn[i, h] = e @ v[keys, kv] / e.sum()
    o = mv("attn_output.weight", attn.astype(np.float32).ravel(), H, nh * hd)
    h2 = oracle.add(x.ravel(), o)
    nf = oracle.rmsnorm(h2, packed["ffn_norm.weight"], H, n)
    act = oracle.swiglu(mv("ffn_gate.weight", nf, S.ffn, H), mv("ffn_up.weight", nf, S.ffn, H))
    return oracle.add(h2, mv("ffn_down.weight", act, H, S.ffn)).reshape(n, H)


# prefill: a code may flip where f16 GEMMs move a key across its border, so the
# reference attends over the rows that the layer stored
@pytest.mark.parametrize("kv,pos,n,window", [
    ("q4", 0, 2, (0, 0)), ("q4", 0, 130, (0, 0)), ("q4", 37, 16, (0, 0)), ("q4", 200, 70, (64, 3)),
    ("f32", 150, 33, (40, 0)), ("fp8", 90, 8, (16, 2))])
def test_tensor_prefill(dev, oracle, weights, kv, pos, n, window):
    oracle.set_fma_mode(False)
    L = Layer.create(dev, weights, FAST.with_(kv=kv, max_keys=512))
    L.set_window(*window)
    L.write_cache(synth.normal(514, "k", pos * KVW), synth.normal(514, "v", pos * KVW))
    x = synth.normal(515, f"p{n}", n * S.hidden).astype(np.float32).reshape(n, S.hidden)
    L.encode_prefill(n, x)
    got = L.read_output(n).reshape(n, S.hidden)
    k, v = L.cache_buffers()
    want = _layer_from_rows(oracle, weights, x, k, v, pos, *window)
    e = abs_err_scaled(got - x, want - x)
    print(f"{kv} prefill {n} at {pos}: layer contribution absErrScaled {e:.2e}")
    assert e <= 1e-2
    # then a decode step: the fast bound over the rows both sides hold
    ref = _ref(oracle, weights, kv, 512, window)
    ref.fill_cache(k, v)
    y = synth.normal(515, "dec", S.hidden).astype(np.float32)
    assert abs_err_scaled(L.forward(y), ref.forward(y, 1)) < 1e-5


@pytest.mark.parametrize("kv", ["q4", "f32"])
def test_model_graph_equals_eager_and_windows_change(dev, kv):
    """The decode graph's launches are sized for max_keys, an eager step's too:
    the same tokens and logits; a window set or dropped between steps counts from
    the next one; rewinding and stepping again gives the same bits."""
    m = synth.model(213, n_layers=2, vocab=4096)
    a, b = (Model.create(dev, m, FAST.with_(kv=kv)) for _ in range(2))
    b.decode_mode = "eager"
    ids = synth.uniform_ids(19, "ids", 600, 4096).tolist()
    for M in (a, b):
        M.step(ids)
    plain = a.decode_device(20).tolist()
    assert plain == b.decode_device(20).tolist()
    for M in (a, b):
        M.set_window(100, 4)
        M.rewind(600)
    first = a.logits([plain[0]])
    assert np.array_equal(bits(first), bits(b.logits([plain[0]])))
    for M in (a, b):
        M.rewind(600)
        M.set_window(0)
    full = a.logits([plain[0]])
    assert not np.array_equal(bits(first), bits(full))
    a.rewind(600)
    assert np.array_equal(bits(full), bits(a.logits([plain[0]])))


def test_window_hides_what_it_should(dev, weights):
    """Keys out of the window do not count, whatever they hold."""
    x = synth.normal(516, "x", S.hidden)
    outs = []
    for fill in (1.0, np.inf):
        kc, vc = (synth.normal(517, t, 90 * KVW).reshape(90, KVW) for t in "kv")
        kc[2:60] = fill
        vc[2:60] = np.nan if fill != 1.0 else 0.0
        L = Layer.create(dev, weights, FAST.with_(max_keys=128))
        L.set_window(31, 2)
        L.write_cache(kc, vc)
        outs.append(L.forward(x))
    assert np.isfinite(outs[0]).all() and np.array_equal(bits(outs[0]), bits(outs[1]))


def test_engines_fall_back(dev):
    m = synth.model(214, n_layers=2, vocab=4096)
    q = Model.create(dev, m, FAST.with_(kv="q4"))
    for mode in ("persistent", "stream"):
        q.decode_mode = mode
        assert q.decode_mode == "kernels"
    p = Model.create(dev, m, FAST)
    p.decode_mode = "persistent"
    ids = synth.uniform_ids(20, "ids", 300, 4096).tolist()
    p.step(ids)
    assert p.decode_mode == "persistent"
    p.set_window(64)
    assert p.decode_mode == "kernels"
    g = Model.create(dev, m, FAST)
    g.step(ids)
    g.set_window(64)
    assert p.decode_device(8).tolist() == g.decode_device(8).tolist()
    p.set_window(0)
    assert p.decode_mode == "persistent"
    p.decode_device(4)


def test_model_q4_near_f32(dev):
    """4 bits move the logits by their own rounding (half a step is a sixteenth
    of a block's largest value), not by an error of the path."""
    m = synth.model(211, n_layers=2, vocab=4096)
    a = Model.create(dev, m, FAST.with_(kv="q4"))
    b = Model.create(dev, m, FAST)
    prompt = synth.uniform_ids(18, "prompt", 300, 4096).tolist()
    e = abs_err_scaled(a.logits(prompt), b.logits(prompt))
    print(f"q4 vs f32 cache logits: absErrScaled {e:.2e}")
    assert e <= 0.2


@pytest.mark.parametrize("over", [dict(attention="exact"), dict(prefill="exact")])
def test_exact_kernels_refuse_q4(dev, weights, over):
    with pytest.raises(FlockError) as e:
        Layer.create(dev, weights, FAST.with_(kv="q4", **over))
    assert e.value.code == -8 and "4-bit" in str(e.value)


def test_window_refusals(dev, weights):
    exact = Layer.create(dev, weights, QWEN3_06B.with_(max_keys=32))
    with pytest.raises(FlockError, match="FLOCK_ATTN_FAST"):
        exact.set_window(4)
    L = Layer.create(dev, weights, FAST.with_(max_keys=32))
    for bad in ((-1, 0), (4, -1), (0, 2)):
        with pytest.raises(FlockError, match="window"):
            L.set_window(*bad)
    m = Model.create(dev, synth.model(215, n_layers=2, vocab=4096), QWEN3_06B)
    with pytest.raises(FlockError, match="FLOCK_ATTN_FAST"):
        m.set_window(16)
    assert m.step([1, 2, 3]) >= 0
