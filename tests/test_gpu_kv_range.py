"""Attention over caches whose elements differ by many powers of two, against the
definition in 64 bits, each block of 32 output dimensions by itself: a large value
or key that a query does not see, or gives no weight to, or that lies in other
dimensions, takes nothing from the rest.

Tolerance.  f32 arithmetic on the stored values: with |q| ~ |k| ~ 1 a score of 128
terms is off by less than 2e-6 and a weight by as much of itself; a block's output
is a sum of n <= 700 terms, each off by that and a few 2^-24 of itself: below 1e-5
of the norm of the block's sum of magnitudes (which stands for the output's own
where terms cancel).
"""
import numpy as np
import pytest

from test_gpu_kv import HD, dev, filled, rows, stored, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
N, NKV, HEADS = 700, 2, 4


def reference(q, k, v, pos, window, sinks):
    """(output, sum of the terms' magnitudes), in f64."""
    nq, heads, _ = q.shape
    g = heads // k.shape[1]
    out, mag = np.zeros((nq, heads, HD)), np.zeros((nq, heads, HD))
    for i in range(nq):
        j = np.arange(pos + i + 1)
        if window:
            j = j[(j > pos + i - window) | (j < sinks)]
        for h in range(heads):
            s = k[j, h // g] @ q[i, h].astype(np.float64) / np.sqrt(HD)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ v[j, h // g]
            mag[i, h] = w @ np.abs(v[j, h // g])
    return out, mag


def kept(torch, x, dtype):  # noqa: F811
    """What the cache keeps; a 4-bit one clamps values at 8 * 65504 first."""
    return stored(torch, np.clip(x, -524032, 524032) if dtype == "q4" else x, dtype)


def check(torch, dev, dtype, q, k, v, pos, window=0, sinks=0):  # noqa: F811
    cap = -(-(len(k) + 5) // 16) * 16
    cache = filled(torch, dev, dtype, k, v, cap, garbage=True)
    out = torch.full(q.shape, float("nan"), device="cuda")
    cache.attention(torch.from_numpy(q).cuda(), pos, out, window=window, sinks=sinks)
    got = out.cpu().numpy().astype(np.float64).reshape(*q.shape[:2], 4, 32)
    want, mag = (x.reshape(got.shape) for x in reference(
        q, kept(torch, k, dtype), kept(torch, v, dtype), pos, window, sinks))
    err = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(mag, axis=-1)
    assert err.max() < 1e-5, err.max()   # a NaN fails


def far_score(q, k, j, by):
    """Key j of every head as far against the queries as `by` in the softmax's exponent
    (the queries share a direction)."""
    d = q.mean((0, 1))
    k[j] = -d / (d @ d) * by * np.sqrt(HD)


def few(seed, nq):
    """nq queries around one direction of norm ~ 128^0.5."""
    r = np.random.default_rng(seed)
    return (r.standard_normal(HD) + 0.1 * r.standard_normal((nq, HEADS, HD))).astype(np.float32)


SMALL = (1, 2, 8, 16)   # rows a kv head: twice as many; below k_kv_prompt's


# The large values' key: first, in a later group, the last but one.
@pytest.mark.parametrize("at", [0, 3, 333, N - 2])
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 17, 2.0 ** 27])
@pytest.mark.parametrize("nq", SMALL)
def test_large_values_of_no_weight_in_four_bits(torch, dev, nq, ratio, at):  # noqa: F811
    k, v, q = rows(1, N, NKV, 0.3), rows(2, N, NKV, 1e-3), few(3, nq)
    v[at] *= ratio
    far_score(q, k, at, 60.0)
    check(torch, dev, "q4", q, k, v, N - nq)


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 17, 2.0 ** 27])
@pytest.mark.parametrize("nq", SMALL)
def test_large_values_of_as_much_weight_in_four_bits(torch, dev, nq, ratio):  # noqa: F811
    """A key whose value times weight is about the others'."""
    k, v, q = rows(4, N, NKV, 0.3), rows(5, N, NKV, 1e-3), few(6, nq)
    v[300] *= ratio
    far_score(q, k, 300, np.log(ratio))
    check(torch, dev, "q4", q, k, v, N - nq)


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 17, 2.0 ** 27])
@pytest.mark.parametrize("nq", SMALL)
def test_large_values_in_other_dimensions_in_four_bits(torch, dev, nq, ratio):  # noqa: F811
    """One block of every value is large, one is zero, one small."""
    k, v, q = rows(7, N, NKV, 0.3), rows(8, N, NKV, 1e-2), few(9, nq)
    v[:, :, 32:64] *= ratio
    v[:, :, 64:96] = 0.0
    v[:, :, 96:] *= 1e-2
    v[:, :, 64] = 1e-30   # a zero scale, no magnitude of 0 to divide by
    cap = -(-(N + 5) // 16) * 16
    cache = filled(torch, dev, "q4", k, v, cap, garbage=True)
    out = torch.full(q.shape, float("nan"), device="cuda")
    cache.attention(torch.from_numpy(q).cuda(), N - nq, out)
    got = out.cpu().numpy().astype(np.float64).reshape(nq, HEADS, 4, 32)
    want, mag = (x.reshape(got.shape) for x in reference(
        q, kept(torch, k, "q4"), kept(torch, v, "q4"), N - nq, 0, 0))
    assert (got[:, :, 2] == 0).all()
    for b in (0, 1, 3):
        err = np.linalg.norm((got - want)[:, :, b], axis=-1) / np.linalg.norm(mag[:, :, b], axis=-1)
        assert err.max() < 1e-5, (b, err.max())


@pytest.mark.parametrize("nq", SMALL)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 20), (3, 1)])
def test_many_scales_in_four_bits(torch, dev, nq, window, sinks):  # noqa: F811
    """Values of every size from f16 subnormal scales to the largest, in a window too;
    the outputs' own size is then that of their largest values."""
    k, v, q = rows(10, N, NKV, 0.3), rows(11, N, NKV), few(12, nq)
    v *= 2.0 ** np.random.default_rng(13).integers(-18, 18, (N, NKV, 1)).astype(np.float32)
    check(torch, dev, "q4", q, k, v, N - nq, window, sinks)


# ------------------------------------------------------- many rows (k_kv_prompt)
# 40 and 300 queries of two heads a kv head: one tile of 128 rows, and five (in pairs)
MANY = (40, 300)
WIDE = ("f32", "bf16")


def late(n, nq):
    """A key that the first three quarters of the queries do not see."""
    return n - nq // 4


@pytest.mark.parametrize("dtype,ratio", [(d, 2.0 ** e) for d in WIDE for e in (8, 13, 20, 30, 90)]
                         + [("q4", 2.0 ** e) for e in (8, 13, 17)])
@pytest.mark.parametrize("nq", (8,) + MANY)
def test_large_values_that_some_queries_do_not_see(torch, dev, nq, dtype, ratio):  # noqa: F811
    k, v, q = rows(20, N, NKV), rows(21, N, NKV), rows(22, nq, HEADS)
    v[late(N, nq)] *= ratio
    check(torch, dev, dtype, q, k, v, N - nq)


@pytest.mark.parametrize("dtype,ratio", [(d, 2.0 ** e) for d in WIDE for e in (8, 13, 20, 30, 90)]
                         + [("q4", 2.0 ** e) for e in (8, 13, 27)])
@pytest.mark.parametrize("nq", (8,) + MANY)
@pytest.mark.parametrize("at", [0, 3, 333])
def test_large_values_of_no_weight(torch, dev, nq, at, dtype, ratio):  # noqa: F811
    k, v, q = rows(23, N, NKV, 0.3), rows(24, N, NKV, 1e-3), few(25, nq)
    v[at] *= ratio
    far_score(q, k, at, 100.0)
    check(torch, dev, dtype, q, k, v, N - nq)


@pytest.mark.parametrize("dtype,ratio", [(d, 2.0 ** e) for d in WIDE for e in (8, 13, 20, 30, 90)]
                         + [("q4", 2.0 ** e) for e in (8, 13, 17)])
@pytest.mark.parametrize("nq", (8,) + MANY)
@pytest.mark.parametrize("what", ["block", "column", "half of the keys", "one small key"])
def test_values_of_two_sizes(torch, dev, nq, what, dtype, ratio):  # noqa: F811
    """From position 0: the first queries see few keys."""
    n = max(nq, 200)
    k, v, q = rows(26, n, NKV), rows(27, n, NKV), rows(28, nq, HEADS)
    if what == "block":
        v[:, :, 32:64] *= ratio
    elif what == "column":
        v[:, :, 5] *= ratio
    elif what == "half of the keys":
        v[nq // 2:] *= ratio
    else:
        v[1:] *= ratio
    check(torch, dev, dtype, q, k[:nq], v[:nq], 0)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("ratio", [2.0 ** e for e in (8, 13, 20, 30, 90)])
@pytest.mark.parametrize("nq", (8,) + MANY)
def test_large_keys_that_some_queries_do_not_see(torch, dev, nq, ratio, dtype):  # noqa: F811
    """Where one is seen it has all the weight, or none (scores further apart than
    f32's exponents)."""
    k, v, q = rows(29, N, NKV), rows(30, N, NKV), rows(31, nq, HEADS)
    at = late(N, nq)
    k[at] *= ratio
    s = np.einsum("qhd,khd->qhk", q.astype(np.float64), np.repeat(stored(torch, k, dtype), 2, 1))
    far = np.abs(s[:, :, at]).min() / np.sqrt(HD)
    if far < 200 and ratio > 2 ** 8:   # not by chance: push the others off
        k[at] = ratio * np.sign(q.mean((0, 1)) + 1e-9)
    check(torch, dev, dtype, q[: 3 * nq // 4], k, v, N - nq)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("ratio", [2.0 ** e for e in (8, 13, 20, 30, 90)])
@pytest.mark.parametrize("nq", (8,) + MANY)
def test_large_keys_in_dimensions_that_queries_leave_out(torch, dev, nq, ratio, dtype):  # noqa: F811
    k, v, q = rows(32, N, NKV), rows(33, N, NKV), rows(34, nq, HEADS)
    k[:, :, 77] *= ratio
    q[:, :, 77] = 0.0
    check(torch, dev, dtype, q, k, v, N - nq)


@pytest.mark.parametrize("dtype", WIDE + ("fp8", "q4"))
@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1e-5, 1e4, 1e30, 1e37])
@pytest.mark.parametrize("nq", (8,) + MANY)
def test_queries_of_any_size(torch, dev, nq, scale, dtype):  # noqa: F811
    """Against keys that make up for it as far as their type goes; a query of 0."""
    low, high = dict(f32=(1e-30, 1e30), bf16=(1e-30, 1e30), fp8=(0.05, 100.0), q4=(1e-3, 1e3))[dtype]
    by = np.float32(min(max(1.0 / scale, low), high))
    if scale * by > 10.0:   # scores past where f32 can tell keys apart
        scale = 10.0 / by
    k, v, q = rows(35, N, NKV, by), rows(36, N, NKV), rows(37, nq, HEADS, np.float32(scale))
    q[nq // 2, 1] = 0.0
    check(torch, dev, dtype, q, k, v, N - nq)


@pytest.mark.parametrize("dtype", WIDE + ("fp8", "q4"))
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-7, 1.0])
@pytest.mark.parametrize("nq", (1, 8) + MANY)
def test_keys_of_zero_see_the_mean(torch, dev, nq, scale, dtype):  # noqa: F811
    k, v, q = np.zeros((N, NKV, HD), np.float32), rows(38, N, NKV), rows(39, nq, HEADS, scale)
    check(torch, dev, dtype, q, k, v, N - nq, window=90, sinks=3)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nq", MANY)
def test_what_is_not_finite_stays_with_the_queries_that_see_it(torch, dev, nq, bad, dtype):  # noqa: F811
    at = late(N, nq)
    seen = at - (N - nq)   # the first query that does
    for which in "kv":
        k, v, q = rows(40, N, NKV), rows(41, N, NKV), rows(42, nq, HEADS)
        x = dict(k=k, v=v)
        x[which][at, :, 9] = bad
        cache = filled(torch, dev, dtype, k, v, 704, garbage=True)
        out = torch.full(q.shape, 7.0, device="cuda")
        cache.attention(torch.from_numpy(q).cuda(), N - nq, out)
        got = out.cpu().numpy().astype(np.float64)
        want, mag = reference(q[:seen], kept(torch, k[:at], dtype), kept(torch, v[:at], dtype),
                              N - nq, 0, 0)
        err = np.linalg.norm(got[:seen] - want, axis=-1) / np.linalg.norm(mag, axis=-1)
        assert err.max() < 1e-5
        if which == "v" and np.isnan(bad):
            assert np.isnan(got[seen:, :, 9]).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "q4"))
def test_many_keys_of_two_sizes_in_splits(torch, dev, dtype):  # noqa: F811
    """One tile of rows, many key splits, of which some have outliers."""
    n, nq = 5000, 50
    k, v, q = rows(43, n, NKV), rows(44, n, NKV), rows(45, nq, HEADS)
    v[700] *= 2.0 ** 16
    v[3000:3100, :, 40:50] *= 2.0 ** 10
    k[700] = 0
    far_score(q, k, 700, 0.0)
    check(torch, dev, dtype, q, k, v, n - nq)
    check(torch, dev, dtype, q, k, v, n - nq, window=2500, sinks=720)


@pytest.mark.parametrize("dtype,scale", [("fp8", 1e36), ("q4", 1e36), ("fp8", 1e34), ("q4", 1e33),
                                         ("f32", 1e36), ("bf16", 1e36)])
@pytest.mark.parametrize("nq", (1, 8) + MANY)
def test_queries_near_the_largest_number(torch, dev, nq, dtype, scale):  # noqa: F811
    """Scores so far apart that one key has all the weight, by a margin of 1e-3 of
    them (f32's own error is 1e-6 of the terms'), on any cache."""
    k, v, q = rows(46, N, NKV, 0.05), rows(47, N, NKV), rows(48, nq, HEADS)
    q /= np.abs(q).max()
    q *= np.float32(scale)
    ks = np.repeat(kept(torch, k, dtype), 2, 1)
    s = np.einsum("qhd,khd->qhk", q.astype(np.float64), ks)
    for i in range(nq):
        s[i, :, N - nq + i + 1:] = -np.inf
    best = np.sort(s, -1)
    sure = (best[..., -1] - best[..., -2]) / best[..., -1] > 1e-3
    cache = filled(torch, dev, dtype, k, v, 704, garbage=True)
    out = torch.full(q.shape, float("nan"), device="cuda")
    cache.attention(torch.from_numpy(q).cuda(), N - nq, out)
    got, vs = out.cpu().numpy(), kept(torch, v, dtype)
    assert np.isfinite(got).all() and sure.mean() > 0.8
    for i, h in zip(*np.nonzero(sure)):
        np.testing.assert_allclose(got[i, h], vs[s[i, h].argmax(), h // 2], rtol=1e-5, atol=1e-6)
