"""Model.step_draft reads draft logits that kernels still in flight write: on the
default stream, on a side stream, on one that the caller names.  Deciding on what
the buffer held before would give other tokens."""
import numpy as np
import pytest

from flock_b200 import lib as flib
from flock_b200 import synth
from flock_b200._abi import FLOCK_E_STATE, FlockError
from flock_b200.layer import QWEN3_06B
from flock_b200.model import Model

pytestmark = pytest.mark.gpu

VOCAB = 4096
IDS = [17, 1, 2, 3, 4, 5]
U = np.full(6, 0.5, np.float32)


@pytest.fixture(scope="module")
def model():
    dev = flib.get_device(0)
    m = Model.create(dev, synth.model(216, n_layers=2, vocab=VOCAB),
                     QWEN3_06B.with_(attention="fast", prefill="tensor", max_keys=512))
    m.step(synth.uniform_ids(21, "prompt", 50, VOCAB).tolist())
    yield m
    dev.close()


@pytest.fixture(scope="module")
def logits():
    """(before, after): a draft certain of its tokens, which are refused unless the
    target is as good as certain too; and one that thinks them impossible (a
    probability of e^-20), whose tokens are kept unless they are so to the target."""
    import torch
    before = torch.zeros(5, VOCAB, device="cuda")
    before[torch.arange(5), torch.tensor(IDS[1:])] = 40.0
    after = torch.zeros(5, VOCAB, device="cuda")
    after[torch.arange(5), torch.tensor(IDS[1:])] = -20.0
    return before, after


def _written_late(buffer, after, scratch):
    """`after` into `buffer` behind some 50 ms of kernels on the current stream."""
    for _ in range(100):
        scratch.add_(1.0)
    buffer.copy_(after)


@pytest.mark.parametrize("where", ["default", "side", "named"])
def test_draft_logits_still_being_written(model, logits, where):
    import torch
    before, after = logits
    pos = model.pos

    def step(draft, **kw):
        out = model.step_draft(IDS, draft=draft, u=U, temperature=1.0, **kw)
        model.rewind(pos)
        return out
    torch.cuda.synchronize()
    want = step(after)
    assert want[:5] == IDS[1:] and step(before)[0] != IDS[1]
    scratch = torch.zeros(1 << 28, device="cuda")   # 1 GB: 0.3 ms and more a pass
    side = torch.cuda.Stream()
    for _ in range(2):
        buffer = before.clone()
        torch.cuda.synchronize()
        if where == "default":
            _written_late(buffer, after, scratch)
            got = step(buffer)
        else:
            with torch.cuda.stream(side):
                _written_late(buffer, after, scratch)
                if where == "side":
                    got = step(buffer)
            if where == "named":
                got = step(buffer, stream=side.cuda_stream)
        assert got == want
        torch.cuda.synchronize()


def test_a_stream_under_capture_is_refused(model, logits):
    import torch
    from flock_b200 import _abi
    s = torch.cuda.Stream()
    x = torch.zeros(16, device="cuda")
    pos, g = model.pos, torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        x += 1
        with pytest.raises(FlockError, match="captured") as e:
            _abi.call("flock_model_wait_stream", model.handle, s.cuda_stream)
        assert e.value.code == FLOCK_E_STATE
    g.replay()   # the capture is whole
    torch.cuda.synchronize()
    assert (x == 1).all() and model.pos == pos
