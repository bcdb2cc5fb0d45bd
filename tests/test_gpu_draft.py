"""Drafted decoding on the GPU (Model.step_draft): the cache append, the attention
of several queries, the draft check and the rewind together, as a decode loop
uses them.  Greedy drafting returns plain decoding's tokens whatever is drafted;
sampled drafting agrees with a 64-bit verification of the model's own logits;
refusals leave the model as it was."""
import numpy as np
import pytest

from flock_b200 import lib as flib
from flock_b200 import synth
from flock_b200._abi import FlockError
from flock_b200.layer import QWEN3_06B
from flock_b200.model import Model
from gpu_util import bits

pytestmark = pytest.mark.gpu

VOCAB = 4096
FAST = QWEN3_06B.with_(attention="fast", prefill="tensor", max_keys=1024)


@pytest.fixture(scope="module")
def dev():
    d = flib.get_device(0)
    yield d
    d.close()


@pytest.fixture(scope="module")
def model_data():
    return synth.model(216, n_layers=2, vocab=VOCAB)


def _prompted(dev, data, cfg, n=200):
    m = Model.create(dev, data, cfg)
    first = m.step(synth.uniform_ids(21, "prompt", n, VOCAB).tolist())
    return m, first


# A multi-token step may have f16 GEMM operands where a single token's are f32, so
# the tokens to compare with come from two-row steps whose draft is (almost always)
# wrong.  Steps of other lengths differ from those in f32 rounding, 1e-6 of a logit;
# two of 4096 logits of this spread (about 1) come that near once in 1e4 steps.
@pytest.mark.parametrize("cfg", [FAST.with_(prefill="exact"), FAST, FAST.with_(kv="q4"),
                                 FAST.with_(kv="q4", matvec="fast"), FAST.with_(kv="bf16")])
@pytest.mark.parametrize("window", [(0, 0), (64, 4)])
def test_greedy_drafts_do_not_change_tokens(dev, model_data, cfg, window):
    a, first = _prompted(dev, model_data, cfg)
    a.set_window(*window)
    tokens, pos = [first], a.pos
    for _ in range(12):   # the right continuation, by two-row steps with a wrong draft
        out = a.step_draft([tokens[-1], (tokens[-1] + 1) % VOCAB])
        tokens.append(out[0])
        assert len(out) <= 2 and a.pos == pos + len(out)
        if len(out) == 2:   # the draft was right after all
            tokens.append(out[1])
        pos = a.pos
    # the same tokens with drafts that are right, wrong from some place on, or all wrong
    for right in (0, 1, 3, 6):
        b, first_b = _prompted(dev, model_data, cfg)
        b.set_window(*window)
        assert first_b == first
        got = [first]
        while len(got) < 10:
            nxt = tokens[len(got):len(got) + 6]
            drafts = nxt[:right] + [(t + 7) % VOCAB for t in nxt[right:]]
            out = b.step_draft([got[-1]] + drafts)
            assert out[:-1] == drafts[:len(out) - 1] and len(out) >= min(right, len(nxt)) + 1
            got += out
            assert b.pos == 200 + len(got) - 1
        n = min(len(got), len(tokens))
        assert got[:n] == tokens[:n]
        # device-fed decoding goes on from the token returned last
        at = b.pos
        cont = int(b.decode_device(1)[0])
        b.rewind(at)
        assert b.step([got[-1]]) == cont


def _verify64(target, draft, ids, u, t):
    """(tokens, the distance of every decision from its border), in f64."""
    def soft(x):
        e = np.exp((x.astype(np.float64) - x.max()) / t)
        return e / e.sum()
    margin, kept = 1.0, 0
    for i, x in enumerate(ids):
        p = soft(target[i])
        q = soft(draft[i]) if draft is not None else np.eye(len(p))[x]
        margin = min(margin, abs(u[i] * q[x] - p[x]) / max(p[x], 1e-30))
        if not u[i] * q[x] < p[x]:
            p = np.maximum(p - q, 0)
            p /= p.sum()
            break
        kept += 1
    else:
        p = soft(target[len(ids)])
    c = np.cumsum(p) / p.sum()
    tok = int(np.searchsorted(c, u[len(ids)], side="right"))
    margin = min(margin, np.abs(c - u[len(ids)]).min())
    return list(ids[:kept]) + [tok], margin


@pytest.mark.parametrize("kv", ["f32", "q4"])
@pytest.mark.parametrize("with_logits", [False, True])
def test_sampled_drafts(dev, oracle, model_data, kv, with_logits):
    """Target logits: the hidden rows of the same step through the oracle's norm and
    head, which the device's match to f32 rounding (4096 x 2^-24 of sums below 1e2
    at the worst order, 1e-6 typically): decisions further than 1e-5 of the
    probability from their border, and of the running sum, must agree."""
    import torch
    oracle.set_fma_mode(False)
    m, _ = _prompted(dev, model_data, FAST.with_(kv=kv))
    m.set_window(FAST.max_keys)   # sees every key; steps of any kind use the same attention
    H = FAST.hidden

    def rows(ids):
        pos, n = m.pos, len(ids)
        hidden = np.asarray(m.encode_partial(ids)).ravel()
        m.rewind(pos)
        x = oracle.rmsnorm(hidden, model_data.output_norm, H, n)
        return oracle.matmul_q8_batched(model_data.embd["packed"], x, VOCAB, H, n).reshape(n, VOCAB)

    rng = np.random.default_rng(22)
    sure, lengths = 0, set()
    for case in range(16):
        d, temp = [0, 1, 3, 5][case % 4], [0.05, 0.3, 1.0, 2.0][case // 4]
        ids = rng.integers(0, VOCAB, d + 1)
        for i in range(d):   # likely drafts: the best token after those before it
            ids[i + 1] = int(np.argmax(rows(ids[:i + 2].tolist())[i]))
        pos, target = m.pos, rows(ids.tolist())
        draft = None
        if with_logits and d:
            draft = (target[:d] + rng.standard_normal((d, VOCAB))).astype(np.float32)
        u = rng.random(d + 1).astype(np.float32)
        want, margin = _verify64(target, draft, ids[1:], u, temp)
        on = None if draft is None else torch.from_numpy(draft).cuda()
        got = m.step_draft(ids.tolist(), draft=on, u=u, temperature=temp)
        assert m.pos == pos + len(got)
        m.rewind(pos)
        assert got == m.step_draft(ids.tolist(), draft=on, u=u, temperature=temp)
        if margin > 1e-5:
            sure += 1
            lengths.add(len(got))
            assert got == want, (case, margin)
    assert sure >= 8 and len(lengths) > 1


def test_errors_leave_the_model_as_it_was(dev, model_data):
    m, first = _prompted(dev, model_data, FAST)
    pos = m.pos

    def refused(match, *a, **kw):
        with pytest.raises((FlockError, ValueError), match=match):
            m.step_draft(*a, **kw)
        assert m.pos == pos
    refused("1 ..", [])
    refused("1 ..", list(range(520)))
    refused("out of range", [VOCAB])
    refused("out of range", [1, -1])
    refused("u only", [1, 2], temperature=1.0)
    refused("temperature", [1, 2], u=[0.5, 0.5], temperature=-1.0)
    refused("temperature", [1, 2], u=[0.5, 0.5], temperature=float("nan"))
    refused("numbers", [1, 2], u=[0.5], temperature=1.0)
    refused("device array", [1, 2], u=[0.5, 0.5], temperature=1.0,
            draft=np.zeros((1, VOCAB), np.float32))
    full, _ = _prompted(dev, model_data, FAST.with_(max_keys=204))
    with pytest.raises(FlockError, match="maxKeys"):
        full.step_draft([1, 2, 3, 4, 5])
    assert full.pos == 200 and len(full.step_draft([1, 2, 3, 4])) >= 1
    # the model goes on from where it was
    other, _ = _prompted(dev, model_data, FAST)
    assert np.array_equal(bits(m.logits([first])), bits(other.logits([first])))


def test_no_distribution_is_refused_and_undone(dev, model_data):
    """NaN logits: the step is undone."""
    import copy
    data = copy.copy(model_data)
    data.output_norm = np.asarray(model_data.output_norm).copy()
    data.output_norm[5] = np.nan
    m = Model.create(dev, data, FAST)
    with pytest.raises(FlockError, match="no distribution"):
        m.step_draft([3, 4, 5], u=[0.1, 0.2, 0.3], temperature=1.0)
    assert m.pos == 0
