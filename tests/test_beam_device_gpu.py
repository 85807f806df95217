"""wav2vec2_b200_beam_device between other calls of its context."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import w2v_b200.binding as b
    return b


class Outputs:
    """Output buffers of n utterances, and as much again behind them that must stay as it was."""

    def __init__(self, n, best, cap):
        self.n, self.best, self.cap = n, best, cap
        self.ids = torch.full((2 * n, best, cap), -7, dtype=torch.int32, device="cuda")
        self.n_ids = torch.full((2 * n, best), -7, dtype=torch.int32, device="cuda")
        self.scores = torch.full((2 * n, best), 7.0, dtype=torch.float64, device="cuda")

    def search(self, m, width, stream=0):
        m.beam_device(width, self.best, self.ids.data_ptr(), self.cap, self.n_ids.data_ptr(), self.scores.data_ptr(), stream)

    def untouched(self, first=0):
        return bool((self.ids[first:] == -7).all() and (self.n_ids[first:] == -7).all() and (self.scores[first:] == 7.0).all())

    def host(self):
        torch.cuda.synchronize()
        return self.ids[:self.n].cpu(), self.n_ids[:self.n].cpu(), self.scores[:self.n].cpu()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("other", ["logits", "transcribe", "debug"])
def test_other_forwards_take_the_batch_away(B, model_path, synth, other):
    """A device batch of 2, then a host call of more utterances (or a debug forward) in the same
    buffers: no search until the next device batch, and not a byte in the caller's outputs."""
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    xs = [synth.make_audio(n, 60 + i) for i, n in enumerate([9000, 6000])]
    d = torch.from_numpy(np.concatenate(xs)).cuda()
    torch.cuda.synchronize()
    m.forward_device(d.data_ptr(), [len(x) for x in xs])
    first = Outputs(2, 3, 60)
    first.search(m, 6)
    ref = first.host()
    assert first.untouched(2) and (ref[1][:, 0] >= 0).all()
    host = [synth.make_audio(5000 + 700 * i, i) for i in range(11)]
    if other == "logits":
        m.logits(host)
    elif other == "transcribe":
        m.transcribe_batch(host)
    else:
        m.debug_stages(host[0])
    o = Outputs(2, 3, 60)
    torch.cuda.synchronize()
    with pytest.raises(B.EngineError, match="replaced"):
        o.search(m, 6)
    torch.cuda.synchronize()
    assert o.untouched()
    m.forward_device(d.data_ptr(), [len(x) for x in xs])
    o.search(m, 6)
    assert same(o.host(), ref) and o.untouched(2)
    m.close()


def test_host_batches_alone_leave_nothing_to_search(B, model_path, synth):
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    m.logits([synth.make_audio(5000, 1)])
    o = Outputs(1, 1, 9)
    o.search(m, 4)
    torch.cuda.synchronize()
    assert o.untouched()
    m.close()
