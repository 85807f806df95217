"""w2v_ctc_beam where its sizes end."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_ctc_beam_gpu import Beam, ctc_logits, search


@pytest.fixture(scope="module")
def K(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import w2v_b200.binding as b
    b.lib()
    return b.kernels


def test_nodes_up_to_the_end_of_an_int(K):
    """A stream at its last frames where width x max_frames is just below 2^31: nodes are numbered
    up to the end of an int.  The frames before are skipped by their count in the state (its first
    word); a hypothesis' walk then goes from the newest nodes through all of them to the oldest."""
    width, max_frames = 128, 16777215
    need = K.ctc_beam_state_bytes(1, 4, width, max_frames)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need + (2 << 30):
        pytest.skip("not enough free device memory")
    lg = ctc_logits(np.random.default_rng(8), 3, 4, 0)
    b = Beam.__new__(Beam)                            # (Beam fills the whole state, 50 GB of it)
    b.K, b.blank, b.width, b.best, b.V, b.lens, b.keep = K, 0, width, 6, 4, [3], []
    b.logits = torch.from_numpy(lg).cuda()
    b.starts, b.max_frames, b.cap = np.zeros(1, np.int64), max_frames, 8
    b.state = torch.empty(need, dtype=torch.uint8, device="cuda")
    b.ids = torch.full((1, 6, 8), -7, dtype=torch.int32, device="cuda")
    b.n_ids = torch.full((1, 6), -7, dtype=torch.int32, device="cuda")
    b.scores = torch.zeros(1, 6, dtype=torch.float64, device="cuda")
    b.err = torch.zeros(1, dtype=torch.int32, device="cuda")
    b.call(0, 1)
    frames = b.state[:4].view(torch.int32)
    assert int(frames.item()) == 1
    frames.fill_(max_frames - 2)
    b.call(1, 2, resume=True)
    b.check([lg])
    b.call(2, 1, resume=True)                         # one more than max_frames
    assert b.results() == [[]] and int(b.err.item()) == 2
    del b
    torch.cuda.empty_cache()
