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


def rms(got, ref):
    return float(((got.double() - ref) ** 2).sum().sqrt() / (ref ** 2).sum().sqrt())


# Relative error (root mean square) of fp32 outputs.  A tensor core's running sum is cut towards zero
# behind its 24th bit at each 16 products; on normal inputs that is 1.1e-6, 2.3e-6, 4.5e-6 and 5.6e-6 of
# the result over K 1024, 2112, 4096 and 5120 in one sum, and 5.8e-7 at any K where the sums end every
# 512; beside a residual of twice the size 6.5e-7, 1.3e-6, 2.6e-6 and 3.3e-6, and 6.5e-7 where they end
# every 1024 (simulated in 64 bits).  The bound lies between the two.
NEAR = {EPI_F32: 8e-7, EPI_F32_RESID: 9e-7}


@pytest.mark.parametrize("weights", ["f16", "q8", "q4"])
@pytest.mark.parametrize("epi", [EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("Kd,rank", [(1024, 16), (2112, 16), (4096, 16), (5120, 16), (2112, 128), (5120, 128), (4096, 72)])
def test_adapters_long_sums_keep_their_bits(K, synth, weights, epi, Kd, rank):
    c = Lora(K, synth, Segments([130, 0, 1, 300]), [1, 0, 0, 2], 1024, Kd, rank, 3, weights, epi)
    c.call()
    c.check()
    ref = c.x.double() @ c.w.double().T + c.bias.double()
    for u, a in enumerate([1, 0, 0, 2]):
        rows = c.seg.rows(u)
        ref[rows] += (c.x[rows].double() @ c.la[a].double().T * float(c.scale[a].double())) @ c.lb[a].double().T
    if epi == EPI_F32_RESID:
        ref += c.resid0.double()
    assert rms(c.out[:c.seg.M], ref) < NEAR[epi]


@pytest.mark.parametrize("epi", [EPI_F32, EPI_F32_RESID])
@pytest.mark.parametrize("N,Kd", [(200, 1024), (200, 2112), (48, 4096), (1024, 5120)])
def test_grouped_long_sums_keep_their_bits(K, epi, N, Kd):
    g = torch.Generator(device="cuda").manual_seed(N + Kd)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    seg, group = Segments([130, 0, 1, 300]), [1, 0, 0, 2]
    x, w, b, resid = r(seg.M, Kd).half(), (r(3, N, Kd) / Kd ** 0.5).half(), r(3, N), 2 * r(seg.M, N)
    out, err = torch.empty(seg.M, N, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    which = torch.tensor(group, dtype=torch.int32, device="cuda")
    K.gemm_grouped(x.data_ptr(), Kd, Kd, seg.M, w.data_ptr(), 3, N, out.data_ptr(), N, b.data_ptr(), resid.data_ptr(), N, epi,
                   seg.off.data_ptr(), seg.T.data_ptr(), which.data_ptr(), 4, err.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    ref = torch.cat([x[seg.rows(u)].double() @ w[e].double().T + b[e].double() for u, e in enumerate(group)])
    if epi == EPI_F32_RESID:
        ref += resid.double()
    assert rms(out, ref) < NEAR[epi]


@pytest.mark.parametrize("weights", ["f16", "q8"])
@pytest.mark.parametrize("epi", [EPI_F16, EPI_F32])
@pytest.mark.parametrize("M,n_adapters", [(64, 32), (64, 33), (65, 16), (65, 17), (128, 16), (128, 17), (129, 10), (129, 11)])
def test_both_sides_of_a_block_per_adapter(K, synth, weights, epi, M, n_adapters):
    """The first product gives each adapter blocks of its own while the 64-row blocks times the
    adapters are 32 or fewer: products of 32 and just past it, adapters that no row uses among
    them, all adapters in the last block's single row's neighbourhood or none."""
    lens = [1] * 20 + [M - 41, 1] + [1] * 20
    which = [(7 * i) % n_adapters if i % 5 else -1 for i in range(len(lens))]
    which = [a if a != 3 else 4 for a in which]                       # adapter 3: no row's
    c = Lora(K, synth, Segments(lens), which, 200, 192, 16, n_adapters, weights, epi)
    assert c.seg.M == M
    c.la[3].fill_(float("nan"))
    c.lb[3].fill_(float("inf"))
    c.call()
    c.check()


@pytest.mark.parametrize("rank,Kd", [(72, 2112), (96, 1088), (128, 1088), (40, 1600)])
@pytest.mark.parametrize("M", [15000, 25000])
def test_long_sums_of_large_ranks_on_every_sm(K, synth, rank, Kd, M):
    """Blocks of the first product whose accumulators and totals take all of an SM's tensor memory,
    more of them than SMs; several adapters in turn in some."""
    lens = [700] * 20 + [1] * 40 + [M - 14040]
    c = Lora(K, synth, Segments(lens), [i % 9 - 1 for i in range(len(lens))], 72, Kd, rank, 8, "f16", EPI_F32)
    assert c.seg.M == M
    c.call()
    c.call()
    c.check()
