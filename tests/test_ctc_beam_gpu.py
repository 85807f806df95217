"""CTC prefix beam search on the device (w2v_ctc_beam) against the search on a
table of prefixes in 64 bits: hypotheses equal, scores within 1e-9 (64-bit
logarithms of sums of some hundred terms; a rounding is 2^-53 of the score)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import w2v_b200.binding as b
    b.lib()
    return b.kernels


def st():
    return torch.cuda.current_stream().cuda_stream


def search(logits, blank, width, counts=False):
    """[(tokens, log-probability)] best first.  Candidates are listed as the
    documented order of equal scores has them (stays, then by beam and token)
    and sorted stably.  `counts`: logits of 0 and -inf; whole numbers of paths,
    exact, in the place of probabilities."""
    if counts:
        add, mul, zero, one, low = (lambda a, b: a + b), (lambda a, b: a * b), 0, 1, 0
    else:
        add, mul, zero, one = np.logaddexp, (lambda a, b: a + b), -np.inf, 0.0
    beams, norm = [((), one, zero)], 0.0
    for row in logits:
        x = row.astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
        if x.max() == -np.inf:
            return []
        z = np.log(np.exp(x - x.max()).sum())
        p = [int(v == 0) for v in x] if counts else x - x.max() - z
        norm += z
        new = {}
        for q, b, n in beams:
            new[q] = [mul(add(b, n), p[blank]), mul(n, p[q[-1]]) if q else zero]
        for q, b, n in beams:
            for c in range(len(row)):
                if c == blank:
                    continue
                e = mul(b if q and c == q[-1] else add(b, n), p[c])
                if e == zero:
                    continue
                r = q + (c,)
                if r in new and any(r == k for k, _, _ in beams):
                    new[r][1] = add(new[r][1], e)
                else:
                    new[r] = [zero, e]
        ranked = sorted(((add(*v), q, v) for q, v in new.items()), key=lambda t: -t[0])[:width]
        least = 0 if counts else ranked[0][0] - 1000 * np.log(2.0)
        beams = [(q, v[0], v[1]) for s, q, v in ranked if s != zero and s >= least]
    if counts:
        return [(q, float(np.log(float(b + n)) - norm)) for q, b, n in beams]
    return [(q, float(np.logaddexp(b, n))) for q, b, n in beams]


class Beam:
    """One batch's search: logits of each utterance as numpy arrays."""

    def __init__(self, K, logits, blank, width, n_best, max_frames=None, cap=None):
        self.K, self.blank, self.width, self.best = K, blank, width, n_best
        self.V = logits[0].shape[1]
        self.lens = [len(x) for x in logits]
        self.logits = torch.from_numpy(np.concatenate(logits + [np.zeros((1, self.V), np.float32)])).cuda()
        self.starts = np.concatenate([[0], np.cumsum(self.lens)[:-1]]).astype(np.int64)
        self.max_frames = max_frames or max(max(self.lens), 1)
        self.cap = cap or self.max_frames
        n = len(logits)
        self.state = torch.full((K.ctc_beam_state_bytes(n, self.V, width, self.max_frames),), 255, dtype=torch.uint8, device="cuda")
        self.ids = torch.full((n, n_best, self.cap), -7, dtype=torch.int32, device="cuda")
        self.n_ids = torch.full((n, n_best), -7, dtype=torch.int32, device="cuda")
        self.scores = torch.full((n, n_best), float("nan"), dtype=torch.float64, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.keep = []

    def call(self, first=0, count=None, resume=False, stream=None):
        """Frames first .. first+count of every utterance (those it has)."""
        T = [max(min(t - first, t if count is None else count), 0) for t in self.lens]
        off = torch.from_numpy(self.starts + np.minimum(first, self.lens)).cuda()
        T = torch.tensor(T, dtype=torch.int32, device="cuda")
        self.keep.append((off, T))
        self.K.ctc_beam(self.logits.data_ptr(), off.data_ptr(), T.data_ptr(), len(self.lens), self.V, self.blank, self.width,
                        self.max_frames, resume, self.state.data_ptr(), self.state.numel(), self.best, self.ids.data_ptr(),
                        self.cap, self.n_ids.data_ptr(), self.scores.data_ptr(), self.err.data_ptr(),
                        st() if stream is None else stream)

    def results(self):
        torch.cuda.synchronize()
        ids, n, s = self.ids.cpu().numpy(), self.n_ids.cpu().numpy(), self.scores.cpu().numpy()
        out = []
        for u in range(len(self.lens)):
            hyps = []
            for h in range(self.best):
                assert (ids[u, h, max(n[u, h], 0):] == -1).all()
                if n[u, h] < 0:
                    assert s[u, h] == -np.inf
                    continue
                hyps.append((tuple(ids[u, h, :n[u, h]].tolist()), s[u, h]))
            out.append(hyps)
        return out

    def check(self, logits, counts=False):
        assert int(self.err.item()) == 0
        for u, got in enumerate(self.results()):
            ref = search(logits[u], self.blank, self.width, counts)[: self.best]
            assert [g[0] for g in got] == [r[0] for r in ref], f"utterance {u}"
            for g, r in zip(got, ref):
                assert abs(g[1] - r[1]) <= 1e-9 * (1 + abs(r[1])), (u, g, r)


def ctc_logits(rng, T, V, blank, peak=6.0):
    lg = rng.standard_normal((T, V)).astype(np.float32) * 1.5
    lg[:, blank] += 4.0
    for t in range(T):
        if rng.random() < 0.3:
            lg[t, rng.integers(V)] += peak
    return lg


@pytest.mark.parametrize("V,width,n_best,lens,blank", [
    (32, 16, 4, [60, 0, 1, 33], 0), (32, 1, 1, [80, 5], 0), (2, 5, 5, [40, 1], 0), (3, 8, 8, [50], 1), (32, 2, 2, [70], 31),
    (5, 128, 10, [40, 12], 2), (32, 100, 10, [50, 3], 0), (64, 33, 3, [40], 7), (94, 20, 2, [45, 2], 0), (200, 9, 9, [30], 199),
    (1024, 4, 2, [12], 3), (33, 127, 127, [20], 0), (31, 31, 31, [25], 30), (300, 100, 5, [12], 0),
    (65, 32, 3, [30, 9], 64), (70, 34, 3, [25], 1), (258, 128, 4, [9], 7)])
def test_hypotheses_and_scores(K, V, width, n_best, lens, blank):
    rng = np.random.default_rng(V * 1000 + width)
    logits = [ctc_logits(rng, t, V, blank) for t in lens]
    b = Beam(K, logits, blank, width, n_best)
    b.call()
    b.check(logits)


@pytest.mark.parametrize("scale", [0.05, 1.0, 30.0])
def test_flat_and_sharp_logits(K, scale):
    """From nearly uniform rows to rows whose tokens are e^-100 apart."""
    rng = np.random.default_rng(int(scale * 100))
    logits = [(rng.standard_normal((40, 12)) * scale).astype(np.float32) for _ in range(3)]
    b = Beam(K, logits, 0, 24, 6)
    b.call()
    b.check(logits)


def test_prefixes_reached_again(K):
    """Two tokens and a narrow beam on noise: prefixes drop out and come back while longer ones live on."""
    rng = np.random.default_rng(77)
    for width in (3, 6, 11):
        logits = [(rng.standard_normal((150, 3)) * 1.2).astype(np.float32) for _ in range(6)]
        b = Beam(K, logits, 0, width, width)
        b.call()
        b.check(logits)


def test_many_tokens_share_a_filter_bit(K):
    """Tokens 64 apart share a bit of the child filter: only the walk tells them apart."""
    rng = np.random.default_rng(5)
    lg = np.full((60, 300), -8.0, np.float32)
    for t in range(60):
        lg[t, [0, 5, 69, 133, 197]] = rng.standard_normal(5) * 1.5
    b = Beam(K, [lg], 0, 7, 7)
    b.call()
    b.check([lg])


def test_equal_scores_in_the_documented_order(K):
    """Rows of 0 and -inf: probabilities are whole numbers of paths, and many are equal."""
    rng = np.random.default_rng(12)
    logits = []
    for _ in range(8):
        lg = np.where(rng.random((14, 6)) < 0.5, 0.0, -np.inf).astype(np.float32)
        lg[np.arange(14), rng.integers(0, 6, 14)] = 0.0
        logits.append(lg)
    for width in (1, 3, 10, 40):
        b = Beam(K, logits, 0, width, min(width, 10))
        b.call()
        b.check(logits, counts=True)


def test_masked_tokens_nan_and_infinities(K):
    rng = np.random.default_rng(4)
    a = ctc_logits(rng, 30, 8, 0)
    a[5:9, 3] = -np.inf
    a[11, :] = -np.inf
    a[11, 4] = 0.5                                    # only token 4
    a[13, 2] = np.nan                                 # cannot be emitted
    low = ctc_logits(rng, 30, 8, 0)
    low[:, 5] = np.finfo(np.float32).min
    inf = ctc_logits(rng, 20, 8, 0)
    inf[7, 3] = np.inf                                # certain
    dead = ctc_logits(rng, 20, 8, 0)
    dead[10] = -np.inf                                # emits nothing: no hypothesis
    dead2 = ctc_logits(rng, 20, 8, 0)
    dead2[0] = np.nan
    no_blank = ctc_logits(rng, 25, 8, 0)
    no_blank[:, 0] = -np.inf
    logits = [a, low, inf, dead, dead2, no_blank]
    b = Beam(K, logits, 0, 10, 5)
    b.call()
    b.check(logits)


def test_far_hypotheses_are_dropped(K):
    """Tokens 2^-1000 less likely than the best one leave no hypothesis; those just above it do."""
    lg = np.zeros((1, 3), np.float32)
    lg[0] = [0.0, -690.0, -696.0]                     # ln 2^-1000 = -693.1
    b = Beam(K, [lg], 0, 3, 3)
    b.call()
    (hyps,) = b.results()
    assert [h[0] for h in hyps] == [(), (1,)]
    assert abs(hyps[1][1] + 690.0) < 1e-9


@pytest.mark.parametrize("hop", [1, 7, 64])
def test_frames_in_pieces(K, hop):
    """The same beams whatever the pieces, down to single frames, with streams that end early."""
    rng = np.random.default_rng(hop)
    logits = [ctc_logits(rng, t, 32, 0) for t in (50, 17, 0, 64)]
    whole = Beam(K, logits, 0, 12, 3)
    whole.call()
    parts = Beam(K, logits, 0, 12, 3, max_frames=200)
    for t in range(0, 64, hop):
        parts.call(t, hop, resume=t > 0)
    whole.check(logits)
    a, b = whole.results(), parts.results()
    assert a == b


def test_partial_results_and_a_new_start(K):
    """Hypotheses after each call are those of the frames so far; resume = 0 forgets them."""
    rng = np.random.default_rng(2)
    lg = ctc_logits(rng, 30, 16, 0)
    b = Beam(K, [lg], 0, 8, 2)
    for t in range(0, 30, 10):
        b.call(t, 10, resume=t > 0)
        b.check([lg[:t + 10]])
    b.call(0, 10, resume=False)
    b.check([lg[:10]])


def test_too_many_frames(K):
    """An utterance past max_frames reports it, keeps its state and gives no hypothesis; the others go on."""
    rng = np.random.default_rng(9)
    logits = [ctc_logits(rng, 30, 8, 0), ctc_logits(rng, 12, 8, 0)]
    b = Beam(K, logits, 0, 4, 2, max_frames=20)
    b.call(0, 12)
    first = b.results()
    b.call(12, 18, resume=True)
    got = b.results()
    assert int(b.err.item()) == 2
    assert got[0] == [] and got[1] == first[1]
    b.err.zero_()
    b.call(12, 8, resume=True)
    b.check([logits[0][:20], logits[1]])


def test_state_that_was_not_started(K):
    rng = np.random.default_rng(9)
    lg = ctc_logits(rng, 10, 8, 0)
    b = Beam(K, [lg], 0, 4, 2)
    b.call(resume=True)
    assert b.results() == [[]] and int(b.err.item()) == 2
    b.err.zero_()
    b.call(0, 5)
    b.width = 3                                       # another width than the state was started with
    b.call(5, 5, resume=True)
    assert b.results() == [[]] and int(b.err.item()) == 2


@pytest.mark.parametrize("n_utt,T,V,width,n_best", [(1, 220, 4, 128, 100), (300, 600, 5, 16, 3)])
def test_more_nodes_than_fit_beside_the_search(K, n_utt, T, V, width, n_best):
    """Hypotheses whose nodes are read in several pieces; more utterances than SMs."""
    lg = ctc_logits(np.random.default_rng(12), T, V, 0)
    b = Beam(K, [lg] * n_utt, 0, width, n_best)
    b.call()
    got = b.results()
    ref = search(lg, 0, width)[:n_best]
    assert len(ref) == n_best and len(ref[0][0]) > T // 8
    for hyps in got:
        assert [g[0] for g in hyps] == [r[0] for r in ref]
        assert all(abs(g[1] - r[1]) <= 1e-9 * (1 + abs(r[1])) for g, r in zip(hyps, ref))


def test_short_id_rows(K):
    """n_ids has the whole length, ids the tokens that fit."""
    lg = np.full((12, 4), -9.0, np.float32)
    for t in range(12):
        lg[t, 1 + t % 3] = 5.0
    b = Beam(K, [lg], 0, 3, 1, cap=5)
    b.call()
    torch.cuda.synchronize()
    assert int(b.n_ids[0, 0]) == 12
    assert b.ids[0, 0].tolist() == [1, 2, 3, 1, 2]


def test_without_outputs(K):
    """n_best = 0 advances the beams and writes nothing."""
    rng = np.random.default_rng(6)
    lg = ctc_logits(rng, 20, 8, 0)
    b = Beam(K, [lg], 0, 4, 2)
    b.best = 0
    b.call(0, 15)
    torch.cuda.synchronize()
    assert (b.n_ids == -7).all() and (b.ids == -7).all()
    b.best = 2
    b.call(15, 5, resume=True)
    b.check([lg])


def test_agrees_with_the_host_decoder(K):
    import w2v_b200.binding as B
    rng = np.random.default_rng(31)
    logits = [ctc_logits(rng, int(t), 32, 0) for t in rng.integers(20, 120, 12)]
    b = Beam(K, logits, 0, 10, 1)
    b.call()
    for lg, hyps in zip(logits, b.results()):
        assert list(hyps[0][0]) == B.ctc_beam_search(lg, 0, 10)


def test_captured_and_on_two_streams(K):
    rng = np.random.default_rng(3)
    sets = [[ctc_logits(rng, t, 24, 0) for t in (40, 25)] for _ in range(2)]
    bs = [Beam(K, x, 0, 6, 2) for x in sets]
    torch.cuda.synchronize()
    for b, s in zip(bs, [torch.cuda.Stream() for _ in bs]):
        for _ in range(3):
            b.call(stream=s.cuda_stream)
    for b, x in zip(bs, sets):
        b.check(x)
    b = bs[0]
    off, T = b.keep[-1]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.K.ctc_beam(b.logits.data_ptr(), off.data_ptr(), T.data_ptr(), 2, b.V, 0, 6, b.max_frames, False, b.state.data_ptr(),
                     b.state.numel(), 2, b.ids.data_ptr(), b.cap, b.n_ids.data_ptr(), b.scores.data_ptr(), b.err.data_ptr(), st())
    b.logits[:65].copy_(torch.from_numpy(np.concatenate([x[::-1] for x in sets[0]])))
    g.replay()
    g.replay()
    b.check([x[::-1] for x in sets[0]])


def test_beam_of_a_forward(K, pkg, model_path, synth):
    """wav2vec2_b200_beam_device: the hypotheses of the last forward's logits, on the
    forward's stream; an utterance too short for a frame has the empty one."""
    import w2v_b200.binding as B
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    xs = [synth.make_audio(n, 40 + i) for i, n in enumerate([9000, 300, 14000, 4321])]
    d = torch.from_numpy(np.concatenate(xs)).cuda()
    n, best, width, cap = len(xs), 3, 6, 60
    ids = torch.full((n, best, cap), -7, dtype=torch.int32, device="cuda")
    n_ids = torch.full((n, best), -7, dtype=torch.int32, device="cuda")
    scores = torch.zeros(n, best, dtype=torch.float64, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):                                # (the later forwards are replayed graphs)
        m.forward_device(d.data_ptr(), [len(x) for x in xs], s.cuda_stream)
        m.beam_device(width, best, ids.data_ptr(), cap, n_ids.data_ptr(), scores.data_ptr(), s.cuda_stream)
    torch.cuda.synchronize()
    assert m.n_frames(300) == 0
    for u, lg in enumerate(m.logits(xs)):
        ref = search(lg, m.cfg["pad_id"], width)[:best]
        got = [(tuple(ids[u, h, :int(n_ids[u, h])].tolist()), float(scores[u, h])) for h in range(best) if n_ids[u, h] >= 0]
        assert [g[0] for g in got] == [r[0] for r in ref], u
        assert all(abs(g[1] - r[1]) <= 1e-9 * (1 + abs(r[1])) for g, r in zip(got, ref))
    for bad in ((0, 1), (129, 1), (4, 5), (4, 0)):
        with pytest.raises(B.EngineError):
            m.beam_device(*bad, ids.data_ptr(), cap, n_ids.data_ptr(), scores.data_ptr())
    with pytest.raises(B.EngineError):
        m.beam_device(4, 1, 0, cap, n_ids.data_ptr(), scores.data_ptr())
    m.close()


def test_beam_without_a_batch(K, pkg, model_path, synth):
    """Before any forward, after one of no utterances and after one whose buffers did not fit there is
    nothing to search; utterances without a frame have the empty hypothesis."""
    import w2v_b200.binding as B
    m = B.Model(model_path("tiny", "q8_0", bias_std=0.02, gain_jitter=0.1))
    audio = torch.from_numpy(synth.make_audio(9000, 3)).cuda()
    ids = torch.full((2, 1, 5), -7, dtype=torch.int32, device="cuda")
    n_ids = torch.full((2, 1), -7, dtype=torch.int32, device="cuda")
    scores = torch.full((2, 1), 7.0, dtype=torch.float64, device="cuda")

    def search():
        m.beam_device(4, 1, ids.data_ptr(), 5, n_ids.data_ptr(), scores.data_ptr())
        torch.cuda.synchronize()
        return n_ids.flatten().tolist(), scores.flatten().tolist()

    untouched = [-7, -7], [7.0, 7.0]
    assert search() == untouched
    m.forward_device(audio.data_ptr(), [8000, 300])
    assert search()[0][1] == 0
    n_ids.fill_(-7), scores.fill_(7.0)
    m.forward_device(audio.data_ptr(), [])
    assert search() == untouched
    with pytest.raises(B.EngineError):           # terabytes of activations: refused by the allocator, nothing is launched
        m.forward_device(audio.data_ptr(), [0x7fffffff] * 4096)
    assert search() == untouched
    m.forward_device(audio.data_ptr(), [300, 20])
    assert search() == ([0, 0], [0.0, 0.0]) and (ids == -1).all()
    m.close()


def test_adapters_heads_and_beams_together(K):
    """One batch of utterances in three languages: a shared projection with an adapter for
    each, an output head for each, and the beams over the logits; logits and hypotheses
    against the same in 64 bits (the search on the logits that came out)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    lens, lang = [37, 0, 64, 21, 50], [2, 0, 1, 0, 2]
    M, Kd, H, V, rank = sum(lens), 192, 256, 24, 16
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, w, bias = r(M, Kd).half(), (r(H, Kd) / Kd ** 0.5).half(), r(H)
    la, lb = (r(3, rank, Kd) / Kd ** 0.5).half(), (r(3, H, rank) / rank ** 0.5).half()
    head, hb = (r(3, V, H) * 3 / H ** 0.5).half(), r(3, V)
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)[:-1]]), dtype=torch.int64, device="cuda")
    T, which = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(lang, dtype=torch.int32, device="cuda")
    h = torch.empty(M, H, dtype=torch.float16, device="cuda")
    logits = torch.empty(M, V, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    work = torch.empty(K.lora_workspace_bytes(M, 5, rank), dtype=torch.uint8, device="cuda")
    state = torch.empty(K.ctc_beam_state_bytes(5, V, 8, 64), dtype=torch.uint8, device="cuda")
    ids = torch.empty(5, 2, 64, dtype=torch.int32, device="cuda")
    n_ids, scores = torch.empty(5, 2, dtype=torch.int32, device="cuda"), torch.empty(5, 2, dtype=torch.float64, device="cuda")
    K.gemm_lora(x.data_ptr(), Kd, Kd, M, w.data_ptr(), H, h.data_ptr(), H, bias.data_ptr(), 0, H, 1, la.data_ptr(), lb.data_ptr(), 0,
                3, rank, off.data_ptr(), T.data_ptr(), which.data_ptr(), 5, work.data_ptr(), work.numel(), err.data_ptr(), st())
    K.gemm_grouped(h.data_ptr(), H, H, M, head.data_ptr(), 3, V, logits.data_ptr(), V, hb.data_ptr(), 0, V, 2, off.data_ptr(),
                   T.data_ptr(), which.data_ptr(), 5, err.data_ptr(), st())
    K.ctc_beam(logits.data_ptr(), off.data_ptr(), T.data_ptr(), 5, V, 0, 8, 64, False, state.data_ptr(), state.numel(), 2,
               ids.data_ptr(), 64, n_ids.data_ptr(), scores.data_ptr(), err.data_ptr(), st())
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    at = 0
    for u, (t, e) in enumerate(zip(lens, lang)):
        xs = x[at:at + t].double()
        z = xs @ w.double().T + bias.double() + (xs @ la[e].double().T) @ lb[e].double().T
        z = 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
        ref = z @ head[e].double().T + hb[e].double()
        # h is rounded to fp16 (2^-11) and its products, at most |h| |head|, are summed
        near = 2.0 ** -10 * (z.abs() @ head[e].double().abs().T) + 1e-3
        got = logits[at:at + t].double()
        assert ((got - ref).abs() <= near).all()
        hyps = search(logits[at:at + t].cpu().numpy(), 0, 8)[:2]
        assert [tuple(ids[u, i, :int(n_ids[u, i])].tolist()) for i in range(len(hyps))] == [q[0] for q in hyps]
        assert all(abs(float(scores[u, i]) - q[1]) <= 1e-9 * (1 + abs(q[1])) for i, q in enumerate(hyps))
        at += t
