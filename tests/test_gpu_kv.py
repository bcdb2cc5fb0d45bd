"""flock_kv_*: caches in caller-owned device memory, against the operators'
definitions in 64 bits (numpy), at the sizes and masks where they can go wrong.

Tolerances.  Append and read are exact.  Attention: scores and outputs are f32
sums of at most 32-bit rounded terms; with |q|, |k| ~ 1 a score of 128 terms
carries about 128^0.5 * 2^-24 * |q||k| < 2e-6 absolute, which moves a weight by
2e-6 relative, and the weighted sum adds n^0.5 2^-24 < 2e-6 relative for the
n <= 5000 keys here: 1e-5 of the output's 2-norm and 1e-4 of its largest entry
hold with a factor of several to spare.
"""
import numpy as np
import pytest

from flock_b200 import lib as flib

pytestmark = pytest.mark.gpu

HD = 128
DTYPES = ("f32", "bf16", "fp8", "q4")


@pytest.fixture(scope="module")
def dev():
    return flib.get_device(0)


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.set_device(0)
    return torch


def q4_values(x):
    """Rows [n][heads][128] as the host's 4-bit quantiser stores them, f64."""
    n, heads, _ = x.shape
    packed = flib.quant_matrix_q4(x.reshape(n * heads, HD), n * heads, HD).reshape(-1, 18)
    d = packed[:, :2].copy().view(np.float16).astype(np.float64)
    q = packed[:, 2:]
    codes = np.concatenate([q & 15, q >> 4], 1).astype(np.float64) - 8
    return (codes * d).reshape(n, heads, HD)


def stored(torch, x, dtype):
    """What the cache keeps of f32 rows, in f64."""
    if dtype == "q4":
        return q4_values(x)
    t = torch.from_numpy(x)
    if dtype == "bf16":
        t = t.to(torch.bfloat16)
    elif dtype == "fp8":
        t = t.clamp(-448, 448).to(torch.float8_e4m3fn)
    return t.to(torch.float32).numpy().astype(np.float64)


def reference(q, k, v, pos, window, sinks):
    """The definition, one query and head at a time, in f64."""
    nq, heads, _ = q.shape
    g = heads // k.shape[1]
    out = np.zeros((nq, heads, HD))
    for i in range(nq):
        p = pos + i
        j = np.arange(p + 1)
        if window:
            j = j[(j > p - window) | (j < sinks)]
        for h in range(heads):
            s = k[j, h // g] @ q[i, h].astype(np.float64) / np.sqrt(HD)
            w = np.exp(s - s.max())
            out[i, h] = (w / w.sum()) @ v[j, h // g]
    return out


def rows(seed, n, heads, scale=1.0):
    return (np.random.default_rng(seed).standard_normal((n, heads, HD)) * scale).astype(np.float32)


def filled(torch, dev, dtype, k, v, capacity, garbage=False):
    from flock_b200.kv import KVCache
    n, nkv, _ = k.shape
    planes = ()
    if garbage:  # planes full of NaN patterns: what no query sees must not matter
        if dtype == "q4":
            planes = [torch.full((nkv, capacity, 64), 0xFF, dtype=torch.uint8, device="cuda")
                      for _ in range(2)]
            planes += [torch.full((nkv, capacity, 4), float("nan"), dtype=torch.float16,
                                  device="cuda") for _ in range(2)]
        else:
            t = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[dtype]
            planes = [torch.full((capacity, nkv, HD), float("nan"), device="cuda").to(t)
                      for _ in range(2)]
    cache = KVCache(dev, dtype, nkv, capacity, *planes)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), 0)
    return cache


def check(torch, cache, dtype, q, k, v, pos, window, sinks):
    out = torch.full(q.shape, float("nan"), device="cuda")
    cache.attention(torch.from_numpy(q).cuda(), pos, out, window=window, sinks=sinks)
    got = out.cpu().numpy().astype(np.float64)
    want = reference(q, stored(torch, k, dtype), stored(torch, v, dtype), pos, window, sinks)
    err = np.linalg.norm(got - want) / np.linalg.norm(want)
    worst = np.abs(got - want).max() / np.abs(want).max()
    assert err < 1e-5 and worst < 1e-4, (err, worst)


# ---------------------------------------------------------------- append, read
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,nkv,pos", [(1, 1, 0), (1, 8, 31), (7, 3, 16), (130, 2, 5)])
def test_append_stores_the_rounded_rows(torch, dev, dtype, n, nkv, pos):
    from flock_b200.kv import KVCache
    cap = -(-(pos + n + 3) // 16) * 16
    cache = KVCache(dev, dtype, nkv, cap)
    before = rows(1, cap, nkv)
    cache.append(torch.from_numpy(before).cuda(), torch.from_numpy(before * 2).cuda(), 0)
    k, v = rows(2, n, nkv, 3.0), rows(3, n, nkv, 0.01)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), pos)
    ko, vo = (torch.empty(cap, nkv, HD, device="cuda") for _ in range(2))
    cache.read(0, cap, ko, vo)
    for got, new, old in ((ko, k, before), (vo, v, before * 2)):
        want = stored(torch, old, dtype)
        want[pos:pos + n] = stored(torch, new, dtype)  # the rows around stay as they were
        np.testing.assert_array_equal(got.cpu().numpy().astype(np.float64), want)


def test_append_codes_ties_zeros_and_extremes_as_the_host(torch, dev):
    from flock_b200.kv import KVCache
    cases = np.zeros((9, 1, HD), np.float32)
    cases[1] = 1.0                                   # every value the first maximum
    cases[2, 0, ::2], cases[2, 0, 1::2] = 4.0, -4.0  # a tie between signs: the first wins
    cases[3, 0] = np.arange(HD) - 64.0
    cases[4, 0] = (np.arange(HD) % 17 - 8) * 0.5     # codes on their borders
    cases[5, 0] = np.float32(1e-9) * (np.arange(HD) % 5)   # scales below f16's smallest
    cases[6, 0, :32] = -7.9999995
    cases[6, 0, 3] = 8.0
    cases[7, 0] = 3e5 * np.cos(np.arange(HD))
    cases[8, 0, 31], cases[8, 0, 32] = 1.0, -1.0
    cache = KVCache(dev, "q4", 1, 16)
    x = torch.from_numpy(cases).cuda()
    cache.append(x, x, 0)
    ko, vo = (torch.empty(9, 1, HD, device="cuda") for _ in range(2))
    cache.read(0, 9, ko, vo)
    for got in (ko, vo):
        np.testing.assert_array_equal(got.cpu().numpy().astype(np.float64), q4_values(cases))


def test_append_saturates_and_marks_nan_blocks(torch, dev):
    from flock_b200.kv import KVCache
    x = rows(4, 1, 1)
    x[0, 0, 5], x[0, 0, 40], x[0, 0, 70] = np.inf, -1e30, np.nan
    cache = KVCache(dev, "q4", 1, 16)
    t = torch.from_numpy(x).cuda()
    cache.append(t, t, 0)
    ko, vo = (torch.empty(1, 1, HD, device="cuda") for _ in range(2))
    cache.read(0, 1, ko, vo)
    want = q4_values(np.nan_to_num(np.clip(x, -524032, 524032)))
    for got in (ko.cpu().numpy(), vo.cpu().numpy()):
        assert np.isnan(got[0, 0, 64:96]).all()
        for part in (slice(0, 64), slice(96, 128)):
            np.testing.assert_array_equal(got[0, 0, part].astype(np.float64), want[0, 0, part])


def test_append_from_a_fused_projection(torch, dev):
    """k and v as strided views of one [n][(heads + 2 kv heads) * 128] buffer."""
    from flock_b200.kv import KVCache
    nkv, heads, n = 2, 4, 5
    fused = torch.from_numpy(rows(5, n, heads + 2 * nkv)).cuda()
    k, v = fused[:, heads:heads + nkv], fused[:, heads + nkv:]
    cache = KVCache(dev, "q4", nkv, 16)
    cache.append(k, v, 3)
    ko, vo = (torch.empty(n, nkv, HD, device="cuda") for _ in range(2))
    cache.read(3, n, ko, vo)
    np.testing.assert_array_equal(ko.cpu().numpy().astype(np.float64),
                                  q4_values(k.contiguous().cpu().numpy()))
    np.testing.assert_array_equal(vo.cpu().numpy().astype(np.float64),
                                  q4_values(v.contiguous().cpu().numpy()))


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,nkv,nq,pos,window,sinks", [
    (2, 1, 1, 0, 0, 0),         # one key
    (16, 8, 1, 1, 0, 0),
    (16, 8, 1, 15, 0, 0),       # a whole 16-key group, and one key more
    (16, 8, 1, 16, 0, 0),
    (16, 8, 1, 63, 0, 0),
    (16, 8, 1, 319, 0, 0),
    (5, 1, 1, 700, 0, 0),       # odd group
    (8, 8, 1, 129, 0, 0),
    (32, 4, 1, 1000, 0, 0),     # group of 8
    (24, 2, 1, 257, 0, 0),      # group of 12
    (40, 2, 1, 90, 0, 0),       # group of 20
    (16, 8, 1, 4099, 0, 0),
    (4, 2, 1, 100, 1, 0),       # the query's own key only
    (4, 2, 1, 100, 1, 1),
    (4, 2, 1, 3, 50, 4),        # a window past the start
    (4, 2, 1, 64, 64, 0),
    (4, 2, 1, 1000, 64, 4),
    (4, 2, 1, 1000, 100, 900),  # sinks up to the window's edge
    (4, 2, 1, 1000, 100, 901),
    (4, 2, 1, 1000, 100, 5000),
    (6, 2, 2, 0, 0, 0),         # drafts
    (16, 8, 6, 250, 0, 0),
    (16, 8, 9, 77, 33, 3),
    (6, 2, 16, 500, 7, 2),
    (4, 4, 5, 0, 2, 1),
    (16, 8, 17, 300, 0, 0),     # prompts
    (4, 2, 64, 0, 0, 0),
    (4, 2, 65, 63, 0, 0),
    (4, 1, 130, 200, 0, 0),
    (2, 2, 129, 127, 40, 3),
    (6, 2, 200, 11, 130, 20),
    (3, 1, 257, 0, 1, 0),
    (4, 2, 100, 900, 300, 64),
])
def test_attention(torch, dev, dtype, heads, nkv, nq, pos, window, sinks):
    n = pos + nq
    cap = -(-(n + 5) // 16) * 16
    k, v = rows(11, n, nkv), rows(12, n, nkv)
    cache = filled(torch, dev, dtype, k, v, cap, garbage=True)
    check(torch, cache, dtype, rows(13, nq, heads), k, v, pos, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [1, 5, 40])
def test_attention_of_peaked_and_of_large_scores(torch, dev, dtype, nq):
    """Scores up to +-60, the largest early, late and at the query's own key."""
    n, nkv, heads = 600, 2, 4
    k, v = rows(21, n, nkv), rows(22, n, nkv)
    q = rows(23, nq, heads)
    k[3, :], k[590, :] = q[0, :nkv] * 3, q[-1, 2:2 + nkv] * 3
    if dtype == "q4":
        k = q4_values(k).astype(np.float32)  # f64-exact in the cache up to the f16 scale
    cache = filled(torch, dev, dtype, k, v, 640, garbage=True)
    check(torch, cache, dtype, q, k, v, n - nq, 0, 0)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "q4"))
@pytest.mark.parametrize("scale", [1e-4, 300.0])
@pytest.mark.parametrize("nq", [1, 3, 33])
def test_attention_of_small_and_large_values(torch, dev, dtype, scale, nq):
    n, nkv, heads = 300, 2, 4
    k, v = rows(31, n, nkv, 0.02), rows(32, n, nkv, scale)
    v[::7] *= 1e-3
    cache = filled(torch, dev, dtype, k, v, 304, garbage=True)
    check(torch, cache, dtype, rows(33, nq, heads, 20.0), k, v, n - nq, 0, 0)


@pytest.mark.parametrize("dtype", ("f32", "q4"))
def test_attention_with_nothing_finite_outside_the_window(torch, dev, dtype):
    """Keys and values that no query sees are NaN and infinite."""
    n, nkv, heads, window, sinks = 500, 2, 4, 60, 3
    k, v = rows(41, n, nkv), rows(42, n, nkv)
    for nq in (1, 4, 30):
        lo = n - nq - window + 1
        kk, vv = k.copy(), v.copy()
        kk[sinks:lo], vv[sinks:lo] = np.nan, np.inf
        if dtype == "q4":
            vv[sinks:lo] = np.nan
        cache = filled(torch, dev, dtype, kk, vv, 512, garbage=True)
        check(torch, cache, dtype, rows(43, nq, heads), k, v, n - nq, window, sinks)


def test_attention_from_and_into_strided_rows(torch, dev):
    nkv, heads, nq, pos = 2, 4, 7, 90
    k, v = rows(51, pos + nq, nkv), rows(52, pos + nq, nkv)
    cache = filled(torch, dev, "q4", k, v, 112)
    q = rows(53, nq, heads)
    fused = torch.zeros(nq, heads + 2 * nkv, HD, device="cuda")
    fused[:, :heads] = torch.from_numpy(q).cuda()
    wide = torch.full((nq, heads + 1, HD), 7.0, device="cuda")
    cache.attention(fused[:, :heads], pos, wide[:, :heads])
    dense = torch.empty(nq, heads, HD, device="cuda")
    cache.attention(torch.from_numpy(q).cuda(), pos, dense)
    assert torch.equal(wide[:, :heads], dense)
    assert (wide[:, heads] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_is_the_same_again_and_on_a_side_stream_and_in_a_graph(torch, dev, dtype):
    nkv, heads, n = 8, 16, 3000
    k, v = rows(61, n, nkv), rows(62, n, nkv)
    cache = filled(torch, dev, dtype, k, v, 3008)
    for nq in (1, 6, 70):
        q = torch.from_numpy(rows(63, nq, heads)).cuda()
        first, again, graphed = (torch.empty_like(q) for _ in range(3))
        cache.attention(q, n - nq, first)
        cache.attention(q, n - nq, again)
        assert torch.equal(first, again)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            again.zero_()
            cache.attention(q, n - nq, again, stream=s.cuda_stream)
        s.synchronize()
        assert torch.equal(first, again)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cache.attention(q, n - nq, graphed, stream=s.cuda_stream)
        for _ in range(3):
            graphed.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(first, graphed)


def test_two_caches_on_two_streams_at_once(torch, dev):
    """Each handle has its own workspace: their calls may overlap."""
    nkv, heads, n = 2, 8, 6000
    k, v = rows(71, n, nkv), rows(72, n, nkv)
    caches = [filled(torch, dev, "q4", k, v, 6000) for _ in range(2)]
    q = torch.from_numpy(rows(73, 1, heads)).cuda()
    want = torch.empty_like(q)
    caches[0].attention(q, n - 1, want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(50)] for _ in range(2)]
    for i in range(50):
        for c, s, o in zip(caches, streams, outs):
            c.attention(q, n - 1, o[i], stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for o in outs for x in o)


def test_no_queries_and_no_rows_are_no_work(torch, dev):
    from flock_b200.kv import KVCache
    cache = KVCache(dev, "q4", 2, 32)
    empty = torch.empty(0, 2, HD, device="cuda")
    cache.append(empty, empty, 32)
    cache.read(32, 0, empty, empty)
    cache.attention(torch.empty(0, 4, HD, device="cuda"), 32, torch.empty(0, 4, HD, device="cuda"))


def test_planes_past_32_bit_offsets(torch, dev):
    """The last keys of a cache whose byte offsets pass 2^32."""
    from flock_b200.kv import KVCache
    nkv, cap = 2, 9_000_000
    k, v = rows(81, 40, nkv), rows(82, 40, nkv)
    for dtype, c in (("q4", cap * 4), ("bf16", cap)):
        cache = KVCache(dev, dtype, nkv, c)
        pos = c - 40
        cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), pos)
        q = rows(83, 40, 4)
        for nq in (1, 40):
            out = torch.empty(nq, 4, HD, device="cuda")
            cache.attention(torch.from_numpy(q[-nq:].copy()).cuda(), c - nq, out, window=1)
            want = np.repeat(stored(torch, v, dtype)[-nq:], 2, axis=1)  # each query's own value
            np.testing.assert_allclose(out.cpu().numpy(), want, rtol=2e-6, atol=1e-6)
        del cache
        torch.cuda.empty_cache()


# ------------------------------------------------------------------- refusals
def test_refusals(torch, dev):
    from flock_b200._abi import FLOCK_E_ARG, FLOCK_E_STATE, FLOCK_E_UNSUPPORTED, FlockError
    from flock_b200.kv import KVCache

    def refused(code, match, f):
        with pytest.raises(FlockError, match=match) as e:
            f()
        assert e.value.code == code

    refused(FLOCK_E_UNSUPPORTED, "head_dim", lambda: KVCache(dev, "q4", 2, 32, head_dim=64))
    refused(FLOCK_E_ARG, "multiple of 16", lambda: KVCache(dev, "q4", 2, 33))
    refused(FLOCK_E_ARG, "capacity", lambda: KVCache(dev, "f32", 2, 0))
    refused(FLOCK_E_ARG, "n_kv_heads", lambda: KVCache(dev, "f32", 0, 16))
    with pytest.raises(ValueError, match="kv dtype"):
        KVCache(dev, "int3", 2, 32)
    with pytest.raises(ValueError, match="no scales"):
        KVCache(dev, "f32", 2, 32, k_scales=torch.zeros(2, 32, 4, device="cuda"))
    with pytest.raises(ValueError, match="workspace"):
        KVCache(dev, "f32", 2, 32, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="k is"):
        KVCache(dev, "f32", 2, 32, torch.zeros(32, 2, 64, device="cuda"),
                torch.zeros(32, 2, 64, device="cuda"))
    cache = KVCache(dev, "q4", 2, 32)
    q, o = (torch.zeros(2, 4, HD, device="cuda") for _ in range(2))
    refused(FLOCK_E_STATE, "inside a cache", lambda: cache.attention(q, 31, o))
    refused(FLOCK_E_STATE, "inside a cache", lambda: cache.attention(q, -1, o))
    refused(FLOCK_E_ARG, "window", lambda: cache.attention(q, 3, o, window=-1))
    refused(FLOCK_E_ARG, "multiple of n_kv_heads",
            lambda: cache.attention(q[:, :3].contiguous(), 3, o[:, :3].contiguous()))
    kv = torch.zeros(2, 2, HD, device="cuda")
    refused(FLOCK_E_STATE, "inside a cache", lambda: cache.append(kv, kv, 31))
    refused(FLOCK_E_STATE, "inside a cache", lambda: cache.read(31, 2, kv, kv))
    with pytest.raises(ValueError, match="torch.float32"):
        cache.attention(q.half(), 3, o)
    with pytest.raises(ValueError, match="cuda"):
        cache.attention(q.cpu(), 3, o)
    with pytest.raises(ValueError, match="not a device array"):
        cache.attention(q.cpu().numpy(), 3, o)
    with pytest.raises(ValueError, match="rows"):
        cache.attention(q, 3, o[:1])
    with pytest.raises(ValueError, match="strides"):
        cache.attention(q.transpose(0, 1).contiguous().transpose(0, 1), 3, o)
    unaligned = torch.zeros(2 * 4 * HD + 1, device="cuda")[1:].view(2, 4, HD)
    refused(FLOCK_E_ARG, "aligned", lambda: cache.attention(unaligned, 3, o))
    refused(FLOCK_E_ARG, "aligned", lambda: cache.append(unaligned[:, :2], unaligned[:, 2:], 3))


# Row tiles (128 rows of a kv head) that run in pairs, with and without a partner
# or live rows in it: two full tiles, a last tile of few rows, nine tiles (the
# tenth empty), splits of a pair's keys, several heads a kv head.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,n,pos,window,sinks", [
    (2, 1, 128, 0, 0, 0), (4, 2, 70, 900, 0, 0), (2, 1, 577, 3, 0, 0), (8, 2, 259, 150, 0, 0),
    (4, 2, 200, 300, 77, 5), (1, 1, 1100, 0, 33, 0), (3, 1, 43, 2000, 1500, 200),
    (4, 2, 50, 17000, 0, 0), (4, 2, 45, 17000, 16500, 40)])   # one tile, alone, many keys
def test_attention_in_pairs(torch, dev, dtype, heads, kv_heads, n, pos, window, sinks):
    keys = pos + n
    k, v, q = rows(91, keys, kv_heads), rows(92, keys, kv_heads), rows(93, n, heads)
    cache = filled(torch, dev, dtype, k, v, -(-(keys + 5) // 16) * 16, garbage=True)
    check(torch, cache, dtype, q, k, v, pos, window, sinks)
    out = [torch.empty(q.shape, device="cuda") for _ in range(2)]
    for o in out:   # the same bits from call to call
        cache.attention(torch.from_numpy(q).cuda(), pos, o, window=window, sinks=sinks)
    assert torch.equal(*out)


def test_more_rows_than_an_int_are_refused(torch, dev):
    from flock_b200._abi import FLOCK_E_LIMIT
    from flock_b200.kv import KVCache
    cache = KVCache(dev, "f32", 2, 32)
    q = torch.zeros(4, device="cuda")   # refused before anything is read
    rc = cache._attention(cache.handle, q.data_ptr(), 0, 2 << 26, 32, 0, 0, 0, q.data_ptr(), 0, None)
    assert rc == FLOCK_E_LIMIT


def test_a_window_past_32_bits_sees_every_key(torch, dev):
    k, v, q = rows(94, 60, 2), rows(95, 60, 2), rows(96, 3, 4)
    cache = filled(torch, dev, "q4", k, v, 64)
    out = [torch.empty(q.shape, device="cuda") for _ in range(2)]
    for o, w in zip(out, (0, 2 ** 32 + 5)):
        cache.attention(torch.from_numpy(q).cuda(), 57, o, window=w)
    assert torch.equal(*out)


@pytest.mark.parametrize("dtype", ["q4", "bf16"])
def test_pairs_in_two_graphs_at_once(torch, dev, dtype):
    """Two captured prompt steps, a cache (and workspace) each, replayed together
    on two streams, three times; a decode step on a third meanwhile."""
    n, nkv, heads, nq = 700, 2, 4, 300
    k, v, q = rows(97, n, nkv), rows(98, n, nkv), torch.from_numpy(rows(99, nq, heads)).cuda()
    caches = [filled(torch, dev, dtype, k, v, 704) for _ in range(3)]
    want = torch.empty(q.shape, device="cuda")
    caches[0].attention(q, n - nq, want)
    outs = [torch.zeros(q.shape, device="cuda") for _ in range(2)]
    one, first = torch.zeros(1, heads, HD, device="cuda"), torch.zeros(1, heads, HD, device="cuda")
    caches[2].attention(q[-1:], n - 1, first)
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in range(3)], []
    for c, o, st in zip(caches, outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            c.attention(q, n - nq, o, stream=st.cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        caches[2].attention(q[-1:], n - 1, one, stream=streams[2].cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        assert torch.equal(one, first)
