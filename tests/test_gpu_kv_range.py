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


@pytest.mark.parametrize("dtype", WIDE + ("fp8", "q4"))
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-7, 1.0])
@pytest.mark.parametrize("nq", (1, 8) + MANY)
def test_keys_of_zero_see_the_mean(torch, dev, nq, scale, dtype):  # noqa: F811
    k, v, q = np.zeros((N, NKV, HD), np.float32), rows(38, N, NKV), rows(39, nq, HEADS, scale)
    check(torch, dev, dtype, q, k, v, N - nq, window=90, sinks=3)
