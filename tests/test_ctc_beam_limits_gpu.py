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


@pytest.mark.parametrize("V,width", [(40, 5), (33, 32), (94, 33), (94, 100), (192, 9), (193, 9), (200, 100), (400, 20), (400, 128), (1024, 31), (1024, 127)])
def test_tokens_of_equal_probability(K, V, width):
    """Logits on a coarse grid, as 16-bit heads and masked tokens of one value give: single frames,
    whose hypotheses in order are the tokens by value and then by id, the blank's (nothing) before
    tokens as likely as it."""
    rng = np.random.default_rng(V + width)
    logits = [(np.round(rng.standard_normal((1, V)) * 2) / g).astype(np.float32) for g in (1, 4, 64)]
    logits += [np.zeros((1, V), np.float32), np.where(rng.random((1, V)) < 0.05, 1.0, -8.0).astype(np.float32)]
    close = np.full((1, V), -1.0, np.float32)         # neighbours of a number: the same leading bits, other values
    close[0, ::3] = np.nextafter(np.float32(-1), np.float32(0))
    logits.append(close)
    b = Beam(K, logits, 3, width, width)
    b.call()
    b.check(logits)


@pytest.mark.parametrize("V,width", [(94, 20), (200, 34), (1024, 6)])
def test_paths_of_equal_probability_among_many_tokens(K, V, width):
    """Rows of 0 and -inf: whole numbers of paths, most of them equal."""
    rng = np.random.default_rng(V)
    lg = np.where(rng.random((7, V)) < 0.4, 0.0, -np.inf).astype(np.float32)
    lg[np.arange(7), rng.integers(0, V, 7)] = 0.0
    b = Beam(K, [lg], 0, width, width)
    b.call()
    b.check([lg], counts=True)
