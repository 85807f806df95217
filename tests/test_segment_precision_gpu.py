"""How exact the adapters' and grouped products are where magnitudes alone (the
tolerances of test_segment_gemm_gpu.py) would not tell."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_segment_gemm_gpu import EPI_F16, EPI_F16_GELU, EPI_F32, EPI_F32_RESID, Lora, Segments, finish


@pytest.fixture(scope="module")
def K(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import w2v_b200.binding as b
    b.lib()
    return b.kernels


@pytest.mark.parametrize("epi", [EPI_F16, EPI_F16_GELU, EPI_F32])
@pytest.mark.parametrize("weights", ["f16", "q8", "q4"])
@pytest.mark.parametrize("lens,rank", [([1, 0, 3], 8), ([70, 1, 200], 24)])
def test_adapters_whose_ranks_cancel(K, synth, weights, epi, lens, rank):
    """Two ranks nearly equal and of opposite sign behind a projection of zeros: the output
    is a hundredth of s A x, which must not be held in fewer bits than the output takes.

    Tolerance: s A x as value and remainder in fp16 (2^-22 of it and half of fp16's least
    step, 2^-25), times |B|; fp32 accumulation as there (2^-23 of the sum of magnitudes per 16
    products); the output's rounding.  Held in fp16 alone, s A x is off by up to 2^-11."""
    c = Lora(K, synth, Segments(lens), [1, 0, 0], 64, 64, rank, 2, weights, epi, bias=False)
    if c.q:
        c.q[1].zero_()                       # scales
    c.w.zero_()
    c.la[:, 1] = (c.la[:, 0].float() + 0.01 * c.la[:, 2].float()).half()
    c.la[:, 2:] = 0
    c.lb[:, :, 1] = -c.lb[:, :, 0]
    c.call()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    for u, a in enumerate([1, 0, 0]):
        rows = c.seg.rows(u)
        x, A, B, s = c.x[rows].double(), c.la[a].double(), c.lb[a].double(), float(c.scale[a].double())
        t = x @ A.T * s
        bound = (2 * 64 / 16 + 2 * rank / 16 + 8) * 2.0 ** -23 * (x.abs() @ A.abs().T * s) @ B.abs().T
        ref, tol = finish(t @ B.T, bound + (t.abs() * 2.0 ** -22 + 2.0 ** -25) @ B.abs().T, epi, None)
        d = (c.out[rows].double() - ref).abs()
        assert (d <= tol).all(), f"max error {d.max().item()} ({(d / tol).max().item()} of what is allowed)"


@pytest.mark.parametrize("weights,N,Kd,rank,epi,lens", [
    ("f16", 200, 128, 16, EPI_F16, [1] * 30), ("f16", 200, 128, 40, EPI_F32, [1] * 30), ("f16", 1024, 256, 8, EPI_F16_GELU, [300, 7, 260, 90]),
    ("f16", 2304, 768, 64, EPI_F16, [499] * 5), ("f16", 93, 640, 24, EPI_F32_RESID, [70, 1, 200]), ("f16", 1024, 1088, 128, EPI_F32_RESID, [300] * 4),
    ("q8", 200, 128, 16, EPI_F16, [1] * 30), ("q8", 93, 128, 40, EPI_F32, [1] * 30), ("q8", 1024, 256, 8, EPI_F16_GELU, [300, 7, 260, 90]),
    ("q8", 1024, 1088, 64, EPI_F32_RESID, [499] * 5), ("q8", 94, 64, 24, EPI_F32_RESID, [70, 1, 200]), ("q8", 2304, 64, 8, EPI_F16, [700] * 40),
    ("q4", 200, 128, 16, EPI_F16, [1] * 30), ("q4", 94, 128, 40, EPI_F32, [1] * 30), ("q4", 1024, 256, 128, EPI_F16_GELU, [300, 7, 260, 90]),
    ("q4", 1024, 1088, 24, EPI_F32_RESID, [499] * 5)])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_an_infinite_adapter_stays_with_its_utterances(K, synth, weights, N, Kd, rank, epi, lens, value):
    """An infinity or NaN in one adapter's second matrix: the outputs it belongs to (its utterances'
    rows, its column) are no numbers, and every other output has the bits it has with a zero there."""
    which = [(2 * i + 1) % 3 for i in range(len(lens))]
    c = Lora(K, synth, Segments(lens), which, N, Kd, rank, 3, weights, epi)
    places = [(0, rank - 1), (N - 1, 0), (N // 2, rank // 2)]
    for n, k in places:
        c.lb[1, n, k] = 0
    c.call()
    c.check()
    clean = c.out.clone()
    for n, k in places:
        c.lb[1, n, k] = value
    c.call()
    torch.cuda.synchronize()
    assert int(c.err.item()) == 0
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for u, a in enumerate(which):
        if a == 1:
            for n, _ in places:
                hit[c.seg.rows(u), n] = True
    assert hit.any() and not hit.all()
    bits = lambda t: t.view(torch.int16 if t.dtype == torch.float16 else torch.int32)
    assert torch.equal(bits(c.out)[~hit], bits(clean)[~hit])
    assert not torch.isfinite(c.out[hit]).any()
    for n, k in places:                                    # and nothing of it is left in the next call
        c.lb[1, n, k] = 0
    c.call()
    torch.cuda.synchronize()
    assert torch.equal(bits(c.out), bits(clean))
