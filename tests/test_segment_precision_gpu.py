"""How exact the adapters' and grouped products are where magnitudes alone (the
tolerances of test_segment_gemm_gpu.py) would not tell."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_segment_gemm_gpu import EPI_F16, EPI_F16_GELU, EPI_F32, Lora, Segments, finish


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
