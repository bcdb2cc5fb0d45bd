"""flock_verify_draft against its rule in 64 bits, one sequence after the other
(numpy).  Tokens and counts are whole numbers and must be equal: a draw is
decided in f64 on both sides, so two borders differ by about 1e-13 of the
total, and the keep test by 1e-7 of a probability -- with the fixed seeds here
no uniform number lies that near a border (checked: `margin`)."""
import numpy as np
import pytest

from flock_b200 import lib as flib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return flib.get_device(0)


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.set_device(0)
    return torch


@pytest.fixture(scope="module")
def scratch(torch):
    from flock_b200.kv import WORKSPACE_BYTES
    # whatever it holds before a call is of no concern
    return torch.full((WORKSPACE_BYTES,), 0xFF, dtype=torch.uint8, device="cuda")


def dist(row, t):
    z = row.astype(np.float64)
    top = z.max()
    if np.isnan(z).any() or not np.isfinite(top):
        return None
    e = np.exp((z - top) / t)
    return e / e.sum()


def rule(target, draft, ids, u, lens, t):
    n, d1, v = target.shape
    tokens, accepted, margin = np.full((n, d1), -1), np.zeros(n, int), 1.0
    for s in range(n):
        w, r = None, 0
        while True:
            if t == 0:
                w = None
                ok = not np.isnan(target[s, r]).all()
                top = int(np.nanargmax(target[s, r])) if ok else -1
                if r == lens[s] or top != ids[s, r]:
                    break
            else:
                w = dist(target[s, r], t)
                if w is None or r == lens[s]:
                    break
                x = ids[s, r]
                inside = 0 <= x < v
                if draft is None:
                    if inside:
                        margin = min(margin, abs(u[s, r] - w[x]) / max(w[x], 1e-30))
                        if u[s, r] < w[x]:
                            tokens[s, r], r = x, r + 1
                            continue
                        rest = w.copy()
                        rest[x] = 0
                        w = rest if rest.sum() > 0 else w
                    break
                q = dist(draft[s, r], t)
                if q is not None and inside and float(u[s, r]) * q[x] < w[x]:
                    margin = min(margin, abs(float(u[s, r]) * q[x] - w[x]) / w[x])
                    tokens[s, r], r = x, r + 1
                    continue
                if q is None:
                    w = None
                else:
                    rest = np.maximum(w - q, 0)
                    w = rest if rest.sum() > 0 else w
                break
            tokens[s, r], r = ids[s, r], r + 1
        accepted[s] = r
        if t == 0:
            tokens[s, r] = top
        elif w is not None:
            c = np.cumsum(w)
            goal = float(u[s, d1 - 1]) * c[-1]
            margin = min(margin, np.abs(c[:-1][w[1:] > 0] - goal).min(initial=1.0) * 1e5)
            tokens[s, r] = int(np.searchsorted(c, goal, side="right"))
    return tokens, accepted, margin


def inputs(seed, n, d, v, spread=2.5):
    r = np.random.default_rng(seed)
    target = (r.standard_normal((n, d + 1, v)) * spread).astype(np.float32)
    draft = (target[:, :d] * 0.9 + r.standard_normal((n, d, v))).astype(np.float32)
    ids = np.zeros((n, d), np.int32)
    for s in range(n):
        for i in range(d):
            ids[s, i] = r.choice(v, p=dist(draft[s, i], 1.0))
    lens = r.integers(0, d + 1, n).astype(np.int32)
    return target, draft, ids, r.random((n, d + 1)).astype(np.float32), lens


def run(torch, dev, scratch, target, draft, ids, u, lens, t):
    from flock_b200.kv import DraftVerifier
    n, d1, v = target.shape
    c = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    tokens = torch.full((n, d1), 99, dtype=torch.int32, device="cuda")
    accepted = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    DraftVerifier(dev, v, scratch).verify(c(target), c(draft), c(ids), c(u), tokens, accepted,
                                          lens=c(lens), temperature=t)
    return tokens.cpu().numpy(), accepted.cpu().numpy()


def check(torch, dev, scratch, target, draft, ids, u, lens, t):
    full = np.full(len(target), ids.shape[1], np.int32) if lens is None else lens
    want, acc, margin = rule(target, draft, ids, u, full, t)
    assert margin > 1e-6, "this seed puts a uniform number on a border"
    got, got_acc = run(torch, dev, scratch, target, draft, ids, u, lens, t)
    np.testing.assert_array_equal(got_acc, acc)
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("t", [0.0, 0.3, 1.0, 1.7])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("n,d,v", [(1, 0, 1), (1, 1, 1), (1, 1, 2), (3, 4, 7), (5, 3, 33),
                                   (2, 2, 1023), (4, 5, 1025), (3, 8, 4096), (7, 1, 5001),
                                   (2, 3, 16385), (3, 4, 70001)])
def test_verify(torch, dev, scratch, n, d, v, probs, t):
    target, draft, ids, u, lens = inputs(n * 100 + d * 10 + v, n, d, v)
    check(torch, dev, scratch, target, draft if probs else None, ids, u, lens, t)


@pytest.mark.parametrize("probs", [True, False])
def test_verify_the_model_vocabulary(torch, dev, scratch, probs):
    target, draft, ids, u, _ = inputs(5, 2, 4, 151936)
    check(torch, dev, scratch, target, draft if probs else None, ids, u, None, 0.8)


def test_verify_a_vocabulary_past_the_on_chip_cache(torch, dev, scratch):
    target, draft, ids, u, _ = inputs(6, 2, 2, 262145)
    u[:, 0] = 0.999  # refuse: the residual's two rows
    check(torch, dev, scratch, target, draft, ids, u, None, 1.0)
    check(torch, dev, scratch, target, None, ids, u, None, 1.0)


def test_verify_many_drafts(torch, dev, scratch):
    target, draft, ids, u, _ = inputs(7, 1, 512, 40)
    check(torch, dev, scratch, target, target[:, :512].copy(), ids, u * 0.9, None, 1.0)
    ids[0] = target[0, :512].argmax(-1)
    check(torch, dev, scratch, target, None, ids, u, None, 0.0)


def test_drafts_from_the_targets_own_distribution_are_all_kept(torch, dev, scratch):
    target, _, ids, u, _ = inputs(8, 4, 6, 3000)
    got, acc = run(torch, dev, scratch, target, target[:, :6].copy(), ids, u * 0.999, None, 1.0)
    assert (acc == 6).all() and (got[:, :6] == ids).all() and (got[:, 6] >= 0).all()


def test_nothing_left_of_the_residual_draws_from_the_target(torch, dev, scratch):
    """A refusal although p = q (u q = p exactly): every residual is 0."""
    target = np.zeros((1, 2, 8), np.float32)
    u = np.array([[1.0, 0.55]], np.float32)
    got, acc = run(torch, dev, scratch, target, target[:, :1].copy(), np.array([[3]], np.int32), u,
                   None, 1.0)
    assert acc[0] == 0 and got[0].tolist() == [4, -1]
    # and without draft logits where the draft holds all of p
    target[0, 0, :] = -np.inf
    target[0, 0, 3] = 0.0
    got, acc = run(torch, dev, scratch, target, None, np.array([[3]], np.int32), u, None, 1.0)
    assert acc[0] == 0 and got[0].tolist() == [3, -1]


def test_masked_rows_and_rows_without_a_distribution(torch, dev, scratch):
    target, draft, ids, u, _ = inputs(9, 6, 2, 300)
    target[0, :, 10:] = -np.inf                      # a few tokens left
    ids[0] = 12                                      # a masked draft is refused
    target[1, 0, 5] = np.nan
    target[2, 1, :] = -np.inf
    target[3, 2, 7] = np.inf
    draft[4, 0, 3] = np.nan
    ids[5, 0], ids[5, 1] = 300, -1                   # not tokens
    u[:] *= 0.2
    for probs in (draft, None):
        check(torch, dev, scratch, target, probs, ids, u, None, 1.0)
    check(torch, dev, scratch, target, None, ids, u, None, 0.0)


def test_greedy_ties_and_nans(torch, dev, scratch):
    target = np.zeros((3, 2, 5000), np.float32)
    target[0, 0, [4000, 700, 4999]] = 2.0            # the lowest of three maxima
    target[1] = np.nan
    target[2, 0, 0], target[2, 0, 9] = -0.0, 0.0     # one value: the lowest index
    ids = np.array([[700], [0], [0]], np.int32)
    got, acc = run(torch, dev, scratch, target, None, ids, np.zeros((3, 2), np.float32), None, 0.0)
    assert acc.tolist() == [1, 0, 1] and got.tolist() == [[700, 0], [-1, -1], [0, 0]]


def test_rows_past_the_drafts_are_not_read(torch, dev, scratch):
    target, draft, ids, u, _ = inputs(10, 3, 4, 500)
    lens = np.array([0, 2, 4], np.int32)
    clean = run(torch, dev, scratch, target, draft, ids, u, lens, 1.0)
    for s, n in enumerate(lens):
        target[s, n + 1:], draft[s, n:], ids[s, n:] = np.nan, np.nan, -7
    got = run(torch, dev, scratch, target, draft, ids, u, lens, 1.0)
    assert all((a == b).all() for a, b in zip(clean, got))
    over = run(torch, dev, scratch, target[2:], draft[2:], ids[2:], u[2:], lens[2:] + 9, 1.0)
    assert (over[0] == got[0][2:]).all()             # counts are clamped


def test_padded_and_unaligned_rows(torch, dev, scratch):
    from flock_b200.kv import DraftVerifier
    target, draft, ids, u, _ = inputs(11, 2, 3, 777)
    want = run(torch, dev, scratch, target, draft, ids, u, None, 1.0)
    for pad, at in ((3, 0), (23, 1), (7, 4)):
        big = [torch.full((2, rows, 777 + pad), float("nan"), device="cuda") for rows in (4, 3)]
        views = [b[:, :, at:at + 777] if at + 777 <= 777 + pad else b[:, :, :777] for b in big]
        for w, x in zip(views, (target, draft)):
            w.copy_(torch.from_numpy(x))
        tokens = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
        accepted = torch.zeros(2, dtype=torch.int32, device="cuda")
        DraftVerifier(dev, 777, scratch).verify(views[0], views[1], torch.from_numpy(ids).cuda(),
                                                torch.from_numpy(u).cuda(), tokens, accepted)
        assert (tokens.cpu().numpy() == want[0]).all() and (accepted.cpu().numpy() == want[1]).all()


def test_the_next_token_follows_the_targets_distribution(torch, dev, scratch):
    """Drafts from a different distribution, checked: the kept-or-drawn first
    token is distributed as the target (20000 draws over 6 tokens; each count
    within 5 standard deviations, 0.5^0.5 / 20000^0.5 * 5 = 0.018)."""
    n, v = 20000, 6
    r = np.random.default_rng(12)
    t_row, d_row = r.standard_normal(v).astype(np.float32), r.standard_normal(v).astype(np.float32)
    ids = r.choice(v, size=(n, 1), p=dist(d_row, 1.0)).astype(np.int32)
    u = r.random((n, 2)).astype(np.float32)
    target = np.broadcast_to(t_row, (n, 2, v))
    got, _ = run(torch, dev, scratch, target, np.broadcast_to(d_row, (n, 1, v)), ids, u, None, 1.0)
    share = np.bincount(got[:, 0], minlength=v) / n
    assert np.abs(share - dist(t_row, 1.0)).max() < 0.018


def test_verify_in_a_graph_and_on_a_side_stream(torch, dev, scratch):
    from flock_b200.kv import DraftVerifier
    target, draft, ids, u, _ = inputs(13, 3, 4, 9000)
    want = run(torch, dev, scratch, target, draft, ids, u, None, 1.0)
    c = [torch.from_numpy(x).cuda() for x in (target, draft, ids, u)]
    tokens = torch.zeros(3, 5, dtype=torch.int32, device="cuda")
    accepted = torch.zeros(3, dtype=torch.int32, device="cuda")
    verifier = DraftVerifier(dev, 9000, scratch)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        verifier.verify(*c, tokens, accepted, stream=s.cuda_stream)
    for _ in range(3):
        tokens.zero_()
        accepted.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert (tokens.cpu().numpy() == want[0]).all() and (accepted.cpu().numpy() == want[1]).all()


def test_refusals(torch, dev, scratch):
    from flock_b200._abi import FLOCK_E_ARG, FLOCK_E_LIMIT, FlockError
    from flock_b200.kv import DraftVerifier
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    i32 = torch.int32
    verifier = DraftVerifier(dev, 10, scratch)
    good = [z(2, 4, 10), z(2, 3, 10), z(2, 3, t=i32), z(2, 4), z(2, 4, t=i32), z(2, t=i32)]

    def refused(code, match, *args, **kw):
        with pytest.raises(FlockError, match=match) as e:
            verifier.verify(*args, **kw)
        assert e.value.code == code

    refused(FLOCK_E_ARG, "temperature", *good, temperature=-1.0)
    refused(FLOCK_E_ARG, "temperature", *good, temperature=float("nan"))
    refused(FLOCK_E_ARG, "temperature", *good, temperature=float("inf"))
    refused(FLOCK_E_ARG, "temperature", *good, temperature=1e-310)
    refused(FLOCK_E_LIMIT, "n_drafts", z(1, 514, 10), None, z(1, 513, t=i32), z(1, 514),
            z(1, 514, t=i32), z(1, t=i32))
    refused(FLOCK_E_LIMIT, "rows", z(40000, 2, 10), None, z(40000, 1, t=i32), z(40000, 2),
            z(40000, 2, t=i32), z(40000, t=i32))
    for at, bad in ((0, z(2, 4, 9)), (1, z(2, 2, 10)), (3, z(2, 3)), (4, z(2, 3, t=i32)),
                    (2, z(2, 3, t=torch.int64)), (5, z(3, t=i32)), (0, z(2, 4, 10).cpu())):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError):
            verifier.verify(*args)
    with pytest.raises(ValueError, match="workspace"):
        DraftVerifier(dev, 10, z(16, t=torch.uint8))
