"""flock_verify_draft at the ends of its arguments' ranges, against test_gpu_verify's
rule in 64 bits: temperatures so small that a row is its maximum alone, uniform
numbers outside [0, 1) and on borders."""
import numpy as np
import pytest

from test_gpu_verify import check, dev, inputs, run, scratch, torch  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("level", [0.0, 30.0, -30.0, 2e4, -3e7])
@pytest.mark.parametrize("t", [1e-3, 1e-7, 1e-9, 1e-30, 1e-38])
@pytest.mark.parametrize("n,d,v", [(2, 3, 1000), (20, 2, 5001), (1, 2, 151936)])
def test_small_temperatures(torch, dev, scratch, n, d, v, t, level, probs):  # noqa: F811
    """The next token is the argmax of a target row, or of what a refused draft
    leaves of one, and always written.  Logits of one row lie apart by 1 or more
    (whole numbers around the level), 1000 times the largest t here."""
    r = np.random.default_rng(v + n)
    target = np.stack([[r.permutation(v) for _ in range(d + 1)] for _ in range(n)])
    draft = target[:, :d] + 0
    for s in range(n):
        for i in range(d):   # half of the drafts agree
            if (s + i) % 2:
                draft[s, i] = r.permutation(v)
    ids = draft.argmax(-1).astype(np.int32)
    # whole numbers that f32 holds at this level, the row's largest near it
    step = max(1.0, float(np.spacing(np.float32(abs(level)))))
    target, draft = (((x - v) * step + level).astype(np.float32) for x in (target, draft))
    u = r.random((n, d + 1)).astype(np.float32)
    check(torch, dev, scratch, target, draft if probs else None, ids, u, None, t)


@pytest.mark.parametrize("t", [1e3, 1e30, 1e38])
def test_large_temperatures(torch, dev, scratch, t):  # noqa: F811
    """Nearly uniform rows; a logit of -inf stays impossible."""
    target, draft, ids, u, _ = inputs(31, 4, 3, 900)
    target[:, :, 100:300] = -np.inf
    draft[:, :, 200:400] = -np.inf
    ids = r_ids(ids, draft)
    check(torch, dev, scratch, target, draft, ids, u, None, t)
    check(torch, dev, scratch, target, None, ids, u, None, t)


def r_ids(ids, draft):
    """Ids that the draft can have drawn."""
    bad = np.isinf(np.take_along_axis(draft, ids[..., None].astype(int), 2)[..., 0])
    return np.where(bad, 0, ids).astype(np.int32)


def test_logits_wider_apart_than_exponents(torch, dev, scratch):  # noqa: F811
    """Differences over t from 0 past 2^31, 2^52 and f64's range: all but the largest
    logit's probability are 0."""
    target = np.full((6, 1, 700), -np.inf, np.float32)
    for s, far in enumerate((705.0, 2e4, 3e9, 1e15, 1e30, 3e38)):
        target[s, 0, 5], target[s, 0, 300], target[s, 0, 699] = -far, 1.0, -far / 2
    u = np.full((6, 1), 0.7, np.float32)
    for t in (1.0, 1e-3):
        got, _ = run(torch, dev, scratch, target, None, np.zeros((6, 0), np.int32), u, None, t)
        assert got[:, 0].tolist() == [300] * 6


def test_temperatures_out_of_range_are_refused(torch, dev, scratch):  # noqa: F811
    from flock_b200._abi import FLOCK_E_ARG, FlockError
    target, draft, ids, u, _ = inputs(32, 1, 1, 8)
    for t in (9e-39, 1e-300, 2e38, 1e300, -1e-9, float("inf"), float("nan")):
        with pytest.raises(FlockError, match="temperature") as e:
            run(torch, dev, scratch, target, draft, ids, u, None, t)
        assert e.value.code == FLOCK_E_ARG


@pytest.mark.parametrize("n,d,v", [(2, 2, 900), (30, 1, 5001)])
def test_uniform_numbers_outside_their_range(torch, dev, scratch, n, d, v):  # noqa: F811
    """A draw takes what is not in [0, 1) as the nearest number that is, NaN as 0:
    some token is drawn wherever there is a distribution."""
    target, draft, ids, u, _ = inputs(33, n, d, v)
    ends = [(-1e-30, 0.0), (-1.0, 0.0), (-np.inf, 0.0), (np.nan, 0.0), (1.0, 1 - 2.0 ** -24),
            (7.0, 1 - 2.0 ** -24), (np.inf, 1 - 2.0 ** -24)]
    for probs in (draft, None):
        for bad, near in ends:
            got = []
            for last in (bad, near):
                x = u.copy()
                x[:, d] = last
                got.append(run(torch, dev, scratch, target, probs, ids, x, None, 1.0))
            (tok, acc), (want, want_acc) = got
            at = np.arange(n), acc
            assert (acc == want_acc).all() and (tok[at] >= 0).all() and (tok[at] < v).all()
            if near == 0.0:   # the first token of any weight
                np.testing.assert_array_equal(tok, want)
            else:             # the last one, or one before it of less than 2^-24 in all
                assert (tok[at] >= want[at]).all()


@pytest.mark.parametrize("n", [9, 64])
def test_a_draw_on_the_border_of_two_blocks(torch, dev, scratch, n):  # noqa: F811
    """Eight times the same 8192 logits, the last 513 of them -inf: at u = k / 8 the
    goal is a running sum but for its rounding, at the end of a block of a cluster (of
    8 or 16 blocks) whose last warps hold no weight.  One warp draws: the last token
    of weight before the border or the first behind it, the same each time."""
    v, period = 65536, 8192
    for seed in range(12):
        r = np.random.default_rng(seed)
        one = (r.standard_normal((n, 1, period)) * 2).astype(np.float32)
        one[:, :, -513:] = -np.inf
        target = np.tile(one, (1, 1, v // period))
        for k in range(1, 8):
            u = np.full((n, 1), k / 8, np.float32)
            got = [run(torch, dev, scratch, target, None, np.zeros((n, 0), np.int32), u, None,
                       1.0)[0][:, 0] for _ in range(2)]
            np.testing.assert_array_equal(*got)
            assert np.isin(got[0], (period * k - 514, period * k)).all(), (seed, k, got[0])
