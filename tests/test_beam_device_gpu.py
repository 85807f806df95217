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


def test_searches_and_forwards_on_several_streams(B, model_path, synth):
    """Searches of one batch on three streams at once share the context's state buffer, and the
    next forward, on a fourth, its logits: each gives what it gives alone."""
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    batches = []
    for k in range(2):
        xs = [synth.make_audio(30000 - 900 * i, 70 + 13 * k + i) for i in range(6 - 3 * k)]
        batches.append((torch.from_numpy(np.concatenate(xs)).cuda(), [len(x) for x in xs]))
    kinds = [(100, 5), (6, 3), (33, 2)]                       # (width, n best)
    refs = []
    for d, lens in batches:
        refs.append([])
        for width, best in kinds:
            m.forward_device(d.data_ptr(), lens)
            o = Outputs(len(lens), best, 120)
            torch.cuda.synchronize()
            o.search(m, width)
            refs[-1].append(o.host())
    streams = [torch.cuda.Stream() for _ in kinds]
    forward = torch.cuda.Stream()
    outs = [[[Outputs(len(b[1]), best, 120) for _, best in kinds] for b in batches] for _ in range(5)]
    torch.cuda.synchronize()
    for turn in outs:
        for (d, lens), os in zip(batches, turn):
            m.forward_device(d.data_ptr(), lens, forward.cuda_stream)
            done = forward.record_event()
            for s, o, (width, _) in zip(streams, os, kinds):
                s.wait_event(done)
                o.search(m, width, s.cuda_stream)
    torch.cuda.synchronize()
    for turn in outs:
        for os, rs in zip(turn, refs):
            for o, r in zip(os, rs):
                assert same(o.host(), r) and o.untouched(o.n)
    m.close()


def test_not_in_a_captured_stream(B, model_path, synth):
    """A replay would search at addresses and sizes of a batch that is gone; the capture goes on
    without it, and the context searches as before."""
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    x = synth.make_audio(20000, 5)
    d = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    m.forward_device(d.data_ptr(), [len(x)])
    a, b = Outputs(1, 2, 80), Outputs(1, 2, 80)
    other = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    a.search(m, 8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        other += 1
        with pytest.raises(B.EngineError, match="captured"):
            b.search(m, 8, torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert b.untouched() and (other == 1).all()
    b.search(m, 8)
    assert same(a.host(), b.host())
    m.close()


def test_closing_a_context_frees_the_search_state(B, model_path, synth):
    """Contexts that have searched, opened and closed in turn (15 MB of beams each)."""
    path = model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1)
    d = torch.from_numpy(np.concatenate([synth.make_audio(160000, 1)] * 10)).cuda()
    o = Outputs(10, 1, 8)
    free = []
    for _ in range(7):
        m = B.Model(path)
        m.forward_device(d.data_ptr(), [160000] * 10)
        o.search(m, 128)
        torch.cuda.synchronize()
        m.close()
        free.append(torch.cuda.mem_get_info()[0])
    assert free[1] - free[-1] < 30 << 20, free
