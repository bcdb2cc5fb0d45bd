"""Greedy drafting against plain decoding, one token a step, of a model whose
multi-token steps have f32 operands (prefill="exact"): the same tokens, whatever is
drafted.  (With prefill="tensor" a step of several tokens has f16 operands and its
tokens are its own: test_gpu_draft.)

Logits of either way differ by f32 rounding, some 1e-5 of a spread of about 1 over
4096 of them: the first two lie that near in about one step of 1e3 here, and the
seed's steps do not."""
import numpy as np
import pytest

from flock_b200 import lib as flib
from flock_b200 import synth
from flock_b200.layer import QWEN3_06B
from flock_b200.model import Model

pytestmark = pytest.mark.gpu

VOCAB = 4096


@pytest.mark.parametrize("kw", [dict(), dict(window=(64, 4)), dict(attention="exact")])
def test_greedy_drafts_are_plain_decoding(kw):
    kw = dict(kw)
    window = kw.pop("window", None)
    dev = flib.get_device(0)
    data = synth.model(216, n_layers=2, vocab=VOCAB)
    cfg = QWEN3_06B.with_(**{**dict(attention="fast", prefill="exact", max_keys=512), **kw})
    prompt = synth.uniform_ids(21, "prompt", 120, VOCAB).tolist()

    def prompted():
        m = Model.create(dev, data, cfg)
        if window:
            m.set_window(*window)
        return m, m.step(prompt)
    a, first = prompted()
    plain = [first] + [int(t) for t in a.decode_device(24)]
    for right in (0, 1, 4):
        b, got = prompted()
        got = [got]
        while len(got) < 20:
            nxt = plain[len(got):len(got) + 5]
            drafts = nxt[:right] + [(t + 7) % VOCAB for t in nxt[right:]]
            got += b.step_draft([got[-1]] + drafts)
        assert got == plain[:len(got)], right
