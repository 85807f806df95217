"""Low-rank adapters beside a shared projection (w2v_gemm_f16_lora,
w2v_gemm_q_lora) and products grouped by utterance (w2v_gemm_grouped_f16)
against their formulas in 64 bits.

Tolerance, element by element, from the arithmetic: the output's rounding
(fp16: half a step, 2^-11 of the value; fp32: 2^-24), fp32 accumulation (at most
one rounding of 2^-23 of the sum of magnitudes per 16 products, in the
adapter's product too), the intermediate s A x held in fp16 (2^-11 of it for
fp16 outputs, 2^-22 as value and remainder for fp32 ones, and fp16's smallest
half step 2^-25), times the GELU's slope (at most 1.13) and its own 1e-6."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPI_F16, EPI_F16_GELU, EPI_F32, EPI_F32_RESID = 0, 1, 2, 3
Q8_0, Q4_0 = 8, 2


@pytest.fixture(scope="module")
def K(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import w2v_b200.binding as b
    b.lib()
    return b.kernels


def st():
    return torch.cuda.current_stream().cuda_stream


def gelu_t(x):
    return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3)))


def is_f16(epi):
    return epi in (EPI_F16, EPI_F16_GELU)


def finish(z, size, epi, resid):
    """Reference and tolerance of the epilogue's output from the product z and its error bound."""
    if epi == EPI_F16_GELU:
        ref, size = gelu_t(z), 1.13 * size + 1e-6
    elif epi == EPI_F32_RESID:
        ref, size = z + resid.double(), size + 2.0 ** -23 * (z.abs() + resid.double().abs())
    else:
        ref = z
    return ref, size + ref.abs() * (2.0 ** -11 if is_f16(epi) else 2.0 ** -24) + (2.0 ** -25 if is_f16(epi) else 0)


class Segments:
    """Utterances as rows off[u] .. off[u]+T[u], `gap` unused rows after each."""

    def __init__(self, lens, gap=0, tail=0):
        self.lens = list(lens)
        off, at = [], 0
        for t in self.lens:
            off.append(at)
            at += max(t, 0) + gap
        self.starts, self.M = off, at + tail
        self.off = torch.tensor(off, dtype=torch.int64, device="cuda")
        self.T = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def rows(self, u):
        return slice(self.starts[u], self.starts[u] + max(self.lens[u], 0))


class Lora:
    def __init__(self, K, synth, seg, adapter, N, Kd, rank, n_adapters, weights="f16", epi=EPI_F16, lda=None, ldc=None,
                 scale=True, bias=True, seed=0, inplace=False):
        g = torch.Generator(device="cuda").manual_seed(seed + 17 * N + Kd + rank)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.K, self.seg, self.N, self.Kd, self.rank, self.na, self.epi = K, seg, N, Kd, rank, n_adapters, epi
        self.lda, self.ldc, M = lda or Kd, ldc or N, seg.M
        self.x = r(max(M, 1), self.lda).half()
        self.la = (r(n_adapters, rank, Kd) / Kd ** 0.5).half()
        self.lb = (r(n_adapters, N, rank) / rank ** 0.5).half()
        self.scale = (torch.rand(n_adapters, device="cuda", generator=g) + 0.5) if scale else None
        self.bias = r(N) if bias else None
        self.adapter = torch.tensor(adapter, dtype=torch.int32, device="cuda")
        dt = torch.float16 if is_f16(epi) else torch.float32
        self.resid = r(max(M, 1), self.ldc) * 2 if epi == EPI_F32_RESID else None
        self.resid0 = self.resid.clone() if self.resid is not None else None
        self.out = self.resid if inplace else torch.full((max(M, 1) + 3, self.ldc), float("nan"), device="cuda", dtype=dt)
        self.q = None
        if weights == "f16":
            self.w = (r(N, Kd) / Kd ** 0.5).half()
        else:
            gtype = Q8_0 if weights == "q8" else Q4_0
            w = (r(N, Kd) / Kd ** 0.5).cpu().numpy()
            raw = synth.quantize_q8_0(w) if gtype == Q8_0 else synth.quantize_q4_0(w)
            raw = torch.from_numpy(np.frombuffer(raw, np.uint8).copy()).cuda()
            ld = (N + 7) // 8 * 8
            codes = torch.empty(N * Kd // (1 if gtype == Q8_0 else 2), dtype=torch.uint8, device="cuda")
            scales = torch.zeros(Kd // 32, ld, dtype=torch.int16, device="cuda")
            self.w = torch.empty(N, Kd, dtype=torch.float16, device="cuda")
            K.repack_q(raw.data_ptr(), gtype, N, Kd, codes.data_ptr(), scales.data_ptr(), ld, st())
            K.dequant(raw.data_ptr(), gtype, N, Kd, self.w.data_ptr(), st())
            torch.cuda.synchronize()
            self.q = (codes, scales, ld, gtype)
        self.work = torch.full((K.lora_workspace_bytes(M, len(seg.lens), rank),), 255, dtype=torch.uint8, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(self, stream=None):
        p = lambda t: t.data_ptr() if t is not None else 0
        tail = (p(self.bias), p(self.resid), self.ldc, self.epi, p(self.la), p(self.lb), p(self.scale), self.na, self.rank,
                p(self.seg.off), p(self.seg.T), p(self.adapter), len(self.seg.lens), p(self.work), self.work.numel(),
                p(self.err), st() if stream is None else stream)
        if self.q:
            codes, scales, ld, gtype = self.q
            self.K.gemm_q_lora(p(self.x), self.lda, self.Kd, self.seg.M, p(codes), p(scales), ld, gtype, self.N,
                               p(self.out), self.ldc, *tail)
        else:
            self.K.gemm_lora(p(self.x), self.lda, self.Kd, self.seg.M, p(self.w), self.N, p(self.out), self.ldc, *tail)

    def check(self):
        torch.cuda.synchronize()
        assert int(self.err.item()) == 0
        M, N, u2 = self.seg.M, self.N, 2.0 ** -23
        x = self.x[:M, :self.Kd].double()
        z = x @ self.w.double().T
        size = x.abs() @ self.w.double().abs().T
        if self.bias is not None:
            z, size = z + self.bias.double(), size + self.bias.double().abs()
        keep = 2.0 ** -11 if is_f16(self.epi) else 2.0 ** -22
        extra = torch.zeros_like(z)
        for u in range(len(self.seg.lens)):
            a, sl = int(self.adapter[u]), self.seg.rows(u)
            if not 0 <= a < self.na or sl.start == sl.stop:
                continue
            s = float(self.scale[a].double()) if self.scale is not None else 1.0
            A, B = self.la[a].double(), self.lb[a].double()
            t = x[sl] @ A.T * s
            z[sl] += t @ B.T
            tsize = x[sl].abs() @ A.abs().T * s
            size[sl] += tsize @ B.abs().T
            extra[sl] = (t.abs() * keep + 2.0 ** -25) @ B.abs().T
        bound = (2 * self.Kd / 16 + 2 * self.rank / 16 + 8) * u2 * size + extra
        ref, tol = finish(z, bound, self.epi, self.resid0[:M, :N] if self.resid0 is not None else None)
        got = self.out[:M, :N].double()
        assert torch.isfinite(got).all()
        d = (got - ref).abs()
        assert (d <= tol).all(), f"max error {d.max().item()} ({(d / tol).max().item()} of what is allowed)"
        if self.out is not self.resid:
            assert torch.isnan(self.out[M:]).all(), "rows behind the last were written"
            assert torch.isnan(self.out[:M, N:]).all(), "columns behind the last were written"


@pytest.mark.parametrize("weights,epi,N,Kd,rank,lens,adapter", [
    ("f16", EPI_F16, 768, 768, 16, [499, 120, 300], [1, 0, 2]),
    ("f16", EPI_F32, 200, 128, 8, [1], [0]),                                    # one row
    ("f16", EPI_F16, 1024, 64, 16, [1] * 16, [3, 0, 0, 3, 1, -1, 2, 2, 1, 0, 7, 3, 3, 2, 1, 0]),   # single frames, -1 and 7: none
    ("f16", EPI_F32_RESID, 768, 1024, 32, [0, 5, 0, 0, 130, 0], [0, 1, 2, 3, 0, 1]),   # empty utterances
    ("f16", EPI_F16_GELU, 320, 512, 24, [65, 63, 64, 1, 127, 129], [0, 1, 0, 2, 1, 1]),
    ("f16", EPI_F32, 94, 256, 64, [33, 200, 31], [0, 1, 2]),                    # N no multiple of 4
    ("f16", EPI_F16, 94, 256, 40, [33, 200, 31], [2, 1, 0]),
    ("f16", EPI_F32_RESID, 5, 192, 128, [70, 70], [1, 0]),
    ("f16", EPI_F16, 2304, 768, 16, [499] * 9, [0, 1, 2, 3, 3, 2, 1, 0, -1]),   # pair tiles
    ("f16", EPI_F16_GELU, 1024, 768, 72, [1000, 2000, 1500], [0, 3, 1]),
    ("q8", EPI_F16, 768, 768, 16, [499, 120, 300], [1, 0, 2]),
    ("q8", EPI_F32, 200, 128, 8, [1], [0]),
    ("q8", EPI_F16, 1024, 64, 16, [1] * 16, [3, 0, 0, 3, 1, -1, 2, 2, 1, 0, 7, 3, 3, 2, 1, 0]),
    ("q8", EPI_F32_RESID, 768, 1024, 32, [0, 5, 0, 0, 130, 0], [0, 1, 2, 3, 0, 1]),
    ("q8", EPI_F16_GELU, 320, 512, 24, [65, 63, 64, 1, 127, 129], [0, 1, 0, 2, 1, 1]),
    ("q8", EPI_F32, 94, 256, 64, [33, 200, 31], [0, 1, 2]),
    ("q8", EPI_F16, 2304, 768, 40, [499] * 9, [0, 1, 2, 3, 3, 2, 1, 0, -1]),
    ("q4", EPI_F16, 768, 768, 16, [499, 120, 300], [1, 0, 2]),
    ("q4", EPI_F32_RESID, 200, 256, 24, [1, 64, 0, 200], [0, 3, 1, 2]),
    ("q4", EPI_F16_GELU, 1024, 768, 128, [999, 1001, 500], [0, 3, 1]),
    ("q4", EPI_F32, 94, 128, 8, [40, 40], [1, 1])])
def test_lora_formula(K, synth, weights, epi, N, Kd, rank, lens, adapter):
    c = Lora(K, synth, Segments(lens), adapter, N, Kd, rank, 4, weights, epi)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
@pytest.mark.parametrize("lens,gap,tail", [([10, 20, 30], 7, 0), ([1, 1, 1, 1], 64, 300), ([3], 0, 70), ([0, 0], 0, 40), ([], 0, 33)])
def test_rows_of_no_utterance_get_the_projection_alone(K, synth, weights, lens, gap, tail):
    c = Lora(K, synth, Segments(lens, gap, tail), [i % 2 for i in range(len(lens))] , 128, 128, 16, 2, weights, EPI_F32)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8", "q4"])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("N,Kd,lens", [(94, 576, [70, 1]), (320, 1088, [300, 40]), (1024, 2112, [499, 600, 801]), (200, 1024, [3, 64])])
def test_long_sums(K, synth, weights, epi, N, Kd, lens):
    """fp32 outputs over more of K than one tensor-core sum takes, whole and broken sums,
    one and two accumulators beside the running total, adapters' blocks behind the last."""
    c = Lora(K, synth, Segments(lens), [i % 2 for i in range(len(lens))], N, Kd, 24, 2, weights, epi)
    c.call()
    c.check()


@pytest.mark.parametrize("epi", [EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("N,Kd", [(94, 576), (320, 2112), (200, 1024)])
def test_grouped_long_sums(K, epi, N, Kd):
    grouped(K, Segments([300, 1, 129, 64, 500]), [0, 2, 1, 1, 0], 3, N, Kd, epi)


@pytest.mark.parametrize("weights", ["f16", "q8", "q4"])
def test_many_adapters_in_one_tile(K, synth, weights):
    """Single frames of 300 streams with 40 adapters in no order: each row tile has nearly all of them."""
    rng = np.random.default_rng(3)
    c = Lora(K, synth, Segments([1] * 300), rng.integers(-1, 41, 300).tolist(), 256, 192, 16, 40, weights, EPI_F16)
    c.call()
    c.check()


@pytest.mark.parametrize("epi", [EPI_F16, EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("rank,n_adapters,N,lens", [(16, 12, 96, [1] * 40), (8, 15, 200, [3] * 50), (64, 3, 94, [1, 0, 200, 5, 77]),
                                                     (128, 1, 40, [9, 130]), (24, 7, 64, [40] * 9), (72, 2, 1024, [1, 1, 1])])
def test_lora_few_rows(K, synth, rank, n_adapters, N, lens, epi):
    """A wave of tiles or less, both products in one kernel: adapters up to what the tile
    holds, operand tiles in several batches, ranks that end inside a step of 16."""
    c = Lora(K, synth, Segments(lens), [i * 5 % (n_adapters + 1) - 1 for i in range(len(lens))], N, 256, rank, n_adapters, "f16", epi)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
@pytest.mark.parametrize("n_utt,top", [(129, 3), (1500, 3), (400, 40), (3000, 2), (700, 0)])
def test_many_utterances(K, synth, weights, n_utt, top):
    """More utterances than the planning threads, most of them short or empty, some long
    ones among them, the first and last empty."""
    rng = np.random.default_rng(n_utt)
    lens = rng.integers(0, top + 1, n_utt)
    lens[[n_utt // 3, n_utt // 2]] = [513, 130]
    lens[0] = lens[-1] = 0
    c = Lora(K, synth, Segments(lens.tolist(), gap=int(top == 2), tail=9), rng.integers(-1, 9, n_utt).tolist(), 136, 128, 16, 8, weights, EPI_F16)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
def test_large_batch_uses_all_row_blocks(K, synth, weights):
    """Enough rows for the 128-row blocks of the first product, utterance ends anywhere in them,
    more than two adapters in some."""
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 260, 160).tolist()
    lens[40:60] = [7] * 20
    c = Lora(K, synth, Segments(lens), rng.integers(-1, 12, 160).tolist(), 128, 192, 32, 12, weights, EPI_F32)
    assert c.seg.M >= 128 * 148
    c.call()
    c.check()


@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72, 104, 128])
@pytest.mark.parametrize("Kd", [64, 192, 1088])
@pytest.mark.parametrize("lens,n_adapters", [([70, 1, 40], 3), ([30] * 12, 12), ([1000] * 18 + [500, 700], 5)])
def test_ranks_and_depths(K, synth, rank, Kd, lens, n_adapters):
    """Fewer steps of K than the first product has stages and warps, and several rounds of its
    stages; each adapter with blocks of its own (few rows), or two and more in turn."""
    c = Lora(K, synth, Segments(lens), [(5 * i + 1) % n_adapters for i in range(len(lens))], 64, Kd, rank, n_adapters, "f16", EPI_F32)
    c.call()
    c.call()
    c.check()


@pytest.mark.parametrize("weights,epi", [("f16", EPI_F16), ("f16", EPI_F32), ("q8", EPI_F16), ("q8", EPI_F32)])
def test_strides_and_missing_operands(K, synth, weights, epi):
    """Rows of A and C further apart than their widths, no bias, no scale."""
    c = Lora(K, synth, Segments([100, 37]), [1, 0], 200, 192, 16, 2, weights, epi, lda=256, ldc=216, scale=False, bias=False)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
@pytest.mark.parametrize("N,ldc", [(256, 256), (93, 95)])
def test_residual_in_place(K, synth, weights, N, ldc):
    c = Lora(K, synth, Segments([100, 37, 260]), [1, 0, 1], N, 192, 16, 2, weights, EPI_F32_RESID, ldc=ldc, inplace=True)
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
def test_unused_adapters_may_hold_anything(K, synth, weights):
    """An adapter no row uses has no influence, NaN and infinities in it included;
    nor has what the workspace held before."""
    c = Lora(K, synth, Segments([70, 0, 90]), [0, 1, 2], 128, 128, 8, 4, weights, EPI_F16)
    c.la[1].fill_(float("nan"))
    c.lb[3].fill_(float("inf"))
    c.lb[1].fill_(float("nan"))
    c.work.fill_(0x7e)           # fp16 NaN
    c.call()
    c.check()


@pytest.mark.parametrize("weights", ["f16", "q8"])
def test_infinite_row_stays_in_its_row(K, synth, weights):
    """A row with an infinity has no influence on the rows of other utterances in its tile."""
    seg = Segments([1] * 20)
    c = Lora(K, synth, seg, [i % 3 for i in range(20)], 128, 128, 16, 3, weights, EPI_F32)
    c.x[7, 5] = float("inf")
    c.call()
    torch.cuda.synchronize()
    bad = ~torch.isfinite(c.out[:20])
    assert bad[7].any() and not bad[:7].any() and not bad[8:20].any()


@pytest.mark.parametrize("weights", ["f16", "q8"])
def test_two_calls_at_once_and_a_replayed_graph(K, synth, weights):
    """Two streams with a workspace each, then a captured call replayed on changed inputs."""
    cs = [Lora(K, synth, Segments([300, 200, 100]), [0, 1, 2], 512, 512, 16, 3, weights, EPI_F16, seed=s) for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(10):
        for c, s in zip(cs, streams):
            c.call(s.cuda_stream)
    for c in cs:
        c.check()
    c = cs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.call(torch.cuda.current_stream().cuda_stream)
    c.x.mul_(-0.5)
    c.adapter.copy_(torch.tensor([2, -1, 0]))
    c.out.fill_(float("nan"))
    g.replay()
    g.replay()
    c.check()


@pytest.mark.parametrize("weights,N", [("f16", 2304), ("q8", 1024)])
def test_lora_repeated_launches_identical(K, synth, weights, N):
    c = Lora(K, synth, Segments([499] * 32), [i % 8 for i in range(32)], N, 768, 16, 8, weights, EPI_F16)
    c.call()
    torch.cuda.synchronize()
    first = c.out.clone()
    for _ in range(20):
        c.call()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    assert torch.equal(first.view(torch.int16), c.out.view(torch.int16))


def grouped(K, seg, group, n_groups, N, Kd, epi, lda=None, ldc=None, bias=True, seed=0, stream=None):
    g = torch.Generator(device="cuda").manual_seed(seed + N + Kd)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    lda, ldc, M = lda or Kd, ldc or N, seg.M
    x = r(max(M, 1), lda).half()
    w = (r(n_groups, N, Kd) / Kd ** 0.5).half()
    b = r(n_groups, N) if bias else None
    resid = r(max(M, 1), ldc) if epi == EPI_F32_RESID else None
    out = torch.full((M + 3, ldc), float("nan"), device="cuda", dtype=torch.float16 if is_f16(epi) else torch.float32)
    gr = torch.tensor(group, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = lambda t: t.data_ptr() if t is not None else 0
    K.gemm_grouped(p(x), lda, Kd, M, p(w), n_groups, N, p(out), ldc, p(b), p(resid), ldc, epi, p(seg.off), p(seg.T), p(gr),
                   len(seg.lens), p(err), st() if stream is None else stream)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    written = torch.zeros(M + 3, dtype=torch.bool, device="cuda")
    for u in range(len(seg.lens)):
        sl = seg.rows(u)
        if not 0 <= group[u] < n_groups or sl.start == sl.stop:
            continue
        written[sl] = True
        xs, ws = x[sl, :Kd].double(), w[group[u]].double()
        z, size = xs @ ws.T, xs.abs() @ ws.abs().T
        if bias:
            z, size = z + b[group[u]].double(), size + b[group[u]].double().abs()
        ref, tol = finish(z, (Kd / 16 + 8) * 2.0 ** -23 * size, epi, resid[sl, :N] if resid is not None else None)
        d = (out[sl, :N].double() - ref).abs()
        assert (d <= tol).all(), f"utterance {u}: max error {d.max().item()} ({(d / tol).max().item()} of what is allowed)"
    assert torch.isnan(out[~written]).all(), "rows of no group were written"
    assert torch.isnan(out[:, N:]).all(), "columns behind the last were written"


@pytest.mark.parametrize("epi", [EPI_F16, EPI_F16_GELU, EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("N,Kd,lens,group,gap", [
    (48, 768, [5, 49, 1, 0, 17], [2, 0, 1, 1, 2], 0),
    (200, 128, [300, 1, 129, 64], [0, 3, 3, 1], 0),
    (94, 64, [1] * 40, [i * 7 % 5 - 1 for i in range(40)], 0),           # groups -1 .. 3 in no order
    (1024, 256, [0, 700, 128, 0, 256, 3], [0, 1, 2, 3, 3, 9], 0),
    (5, 1024, [31, 33, 32], [0, 0, 3], 5),
    (256, 192, [127, 1, 128], [1, 2, 3], 1)])
def test_grouped_formula(K, epi, N, Kd, lens, group, gap):
    grouped(K, Segments(lens, gap, tail=gap), group, 4, N, Kd, epi)


@pytest.mark.parametrize("epi", [EPI_F16, EPI_F32, EPI_F32_RESID])
def test_grouped_strides(K, epi):
    grouped(K, Segments([100, 37], 3), [1, 0], 2, 200, 192, epi, lda=256, ldc=216, bias=False)
    grouped(K, Segments([100, 37], 3), [1, 0], 2, 93, 192, epi, lda=200, ldc=95)


def test_grouped_without_rows(K):
    grouped(K, Segments([0, 0, 0], 0, 5), [0, 1, 0], 2, 64, 64, EPI_F32)
    grouped(K, Segments([], 0, 5), [], 2, 64, 64, EPI_F32)
    grouped(K, Segments([4, 4], 0, 5), [-1, 2], 2, 64, 64, EPI_F32)


def test_grouped_many_utterances(K):
    """More utterances than a warp looks at in one step, most of them short or empty."""
    rng = np.random.default_rng(8)
    lens = rng.integers(0, 4, 700)
    lens[[13, 300, 699]] = [200, 513, 130]
    grouped(K, Segments(lens.tolist()), rng.integers(0, 12, 700).tolist(), 12, 136, 192, EPI_F16)


def test_grouped_infinite_weights_of_other_groups(K):
    """Weights of a group that no row uses, and rows of no utterance, may hold anything."""
    seg = Segments([3, 40], gap=2)
    x = torch.randn(seg.M, 64, device="cuda").half()
    x[3:5] = float("nan")
    w = torch.randn(3, 72, 64, device="cuda").half()
    w[1] = float("inf")
    out = torch.zeros(seg.M, 72, device="cuda")
    gr = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    K.gemm_grouped(x.data_ptr(), 64, 64, seg.M, w.data_ptr(), 3, 72, out.data_ptr(), 72, 0, 0, 0, EPI_F32, seg.off.data_ptr(),
                   seg.T.data_ptr(), gr.data_ptr(), 2, 0, st())
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (out[3:5] == 0).all()


def test_grouped_overlapping_utterances(K):
    """Utterances that claim the same rows are not allowed for; a call that has many of them
    ends, and stays within the rows."""
    M, N, Kd, n = 300, 64, 128, 200
    x, w = torch.randn(M, Kd, device="cuda").half(), (torch.randn(1, N, Kd, device="cuda") / Kd ** 0.5).half()
    out = torch.full((M + 3, N), float("nan"), device="cuda")
    off, T = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.full((n,), M, dtype=torch.int32, device="cuda")
    which, err = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    K.gemm_grouped(x.data_ptr(), Kd, Kd, M, w.data_ptr(), 1, N, out.data_ptr(), N, 0, 0, N, EPI_F32, off.data_ptr(), T.data_ptr(),
                   which.data_ptr(), n, err.data_ptr(), st())
    torch.cuda.synchronize()
    assert int(err.item()) == 0 and torch.isnan(out[M:]).all()
    z, size = x.double() @ w[0].double().T, x.double().abs() @ w[0].double().abs().T
    assert ((out[:M].double() - z).abs() <= (Kd / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -24 * z.abs()).all()
