"""Calls that the adapter, grouped-product and beam-search launchers refuse:
the host checks answer before anything is launched, so no GPU is needed."""
import pytest

OK, ARGS, CAPACITY = 0, 1, 6
P = 4096          # a 16-byte aligned address that is never read


@pytest.fixture(scope="module")
def L(pkg):
    import w2v_b200.binding as b
    return b.lib()


def lora(L, **kw):
    a = dict(A=P, lda=128, K=128, M=10, B=P, N=64, C=P, ldc=64, bias=None, resid=None, ldr=0, epilogue=0, la=P, lb=P, ls=None,
             n_adapters=2, rank=16, off=P, T=P, adapter=P, n_utt=3, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return L.w2v_gemm_f16_lora(*a.values(), None, None)


def lora_q(L, **kw):
    a = dict(A=P, lda=128, K=128, M=10, Bq=P, Bs=P, ld_s=64, gguf_type=8, N=64, C=P, ldc=64, bias=None, resid=None, ldr=0,
             epilogue=0, la=P, lb=P, ls=None, n_adapters=2, rank=16, off=P, T=P, adapter=P, n_utt=3, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return L.w2v_gemm_q_lora(*a.values(), None, None)


BAD = [dict(K=100), dict(K=0), dict(lda=120), dict(lda=132), dict(N=0), dict(ldc=60), dict(M=-1), dict(epilogue=4), dict(epilogue=-1),
       dict(epilogue=3), dict(epilogue=3, resid=P, ldr=60), dict(rank=0), dict(rank=12), dict(rank=136), dict(n_adapters=0), dict(la=None),
       dict(lb=None), dict(la=P + 2), dict(lb=P + 8), dict(A=P + 2), dict(A=None), dict(C=None), dict(off=None), dict(T=None),
       dict(adapter=None), dict(n_utt=-1), dict(ws=None), dict(ws=P + 16)]


@pytest.mark.parametrize("bad", BAD + [dict(B=None), dict(B=P + 4)])
def test_lora_refuses(L, bad):
    assert lora(L, **bad) == ARGS


@pytest.mark.parametrize("bad", BAD + [dict(Bq=None), dict(Bs=None), dict(Bs=P + 2), dict(gguf_type=1), dict(ld_s=56), dict(ld_s=68)])
def test_lora_q_refuses(L, bad):
    assert lora_q(L, **bad) == ARGS


@pytest.mark.parametrize("f", [lora, lora_q])
def test_lora_workspace(L, f):
    need = L.w2v_lora_workspace_bytes(10, 3, 16)
    assert need > 0
    assert f(L, ws_bytes=need - 1) == CAPACITY
    assert f(L, M=0, A=None, C=None) == OK                    # no rows: nothing to do
    for bad in ((-1, 3, 16), (10, -1, 16), (10, 3, 12), (10, 3, 0), (10, 3, 136)):
        assert L.w2v_lora_workspace_bytes(*bad) == -1
    assert L.w2v_lora_workspace_bytes(100000, 4096, 128) > 0


def group(L, **kw):
    a = dict(A=P, lda=128, K=128, M=10, B=P, n_groups=2, N=64, C=P, ldc=64, bias=None, resid=None, ldr=0, epilogue=0, off=P, T=P,
             group=P, n_utt=3)
    a.update(kw)
    return L.w2v_gemm_grouped_f16(*a.values(), None, None)


@pytest.mark.parametrize("bad", [dict(K=100), dict(K=0), dict(lda=120), dict(lda=132), dict(N=0), dict(ldc=60), dict(M=-1), dict(epilogue=4),
                                 dict(epilogue=-1), dict(epilogue=3), dict(n_groups=0), dict(B=None), dict(B=P + 2), dict(A=P + 2),
                                 dict(A=None), dict(C=None), dict(off=None), dict(T=None), dict(group=None), dict(n_utt=-1)])
def test_grouped_refuses(L, bad):
    assert group(L, **bad) == ARGS


def test_grouped_without_rows(L):
    assert group(L, M=0, A=None, C=None) == OK
    assert group(L, n_utt=0, off=None, T=None, group=None) == OK


def beam(L, **kw):
    a = dict(logits=P, off=P, T=P, n_utt=2, V=32, blank=0, width=8, max_frames=100, resume=0, state=P, state_bytes=1 << 40, n_best=2,
             ids=P, cap=100, n_ids=P, scores=P)
    a.update(kw)
    return L.w2v_ctc_beam(*a.values(), None, None)


@pytest.mark.parametrize("bad", [dict(V=1), dict(V=1025), dict(blank=-1), dict(blank=32), dict(width=0), dict(width=129), dict(max_frames=0),
                                 dict(max_frames=1 << 30), dict(n_best=-1), dict(n_best=9), dict(n_utt=-1), dict(logits=None), dict(off=None),
                                 dict(T=None), dict(state=None), dict(state=P + 8), dict(ids=None), dict(n_ids=None), dict(scores=None),
                                 dict(cap=0)])
def test_beam_refuses(L, bad):
    assert beam(L, **bad) == ARGS


def test_beam_state(L):
    need = L.w2v_ctc_beam_state_bytes(2, 32, 8, 100)
    assert need > 0 and L.w2v_ctc_beam_state_bytes(0, 32, 8, 100) == 0
    assert beam(L, state_bytes=need - 1) == CAPACITY
    assert beam(L, n_utt=0, logits=None, off=None, T=None, state=None, state_bytes=0) == OK
    for bad in ((-1, 32, 8, 100), (2, 1, 8, 100), (2, 1025, 8, 100), (2, 32, 0, 100), (2, 32, 129, 100), (2, 32, 8, 0), (2, 32, 128, 1 << 24)):
        assert L.w2v_ctc_beam_state_bytes(*bad) == -1


HUGE = 0x7fffffff - 100          # sizes whose tiles an int could not number


@pytest.mark.parametrize("f", [lora, lora_q, group])
@pytest.mark.parametrize("bad", [dict(M=HUGE), dict(N=HUGE, ldc=HUGE, ld_s=HUGE + 7 & ~7), dict(n_utt=HUGE)])
def test_sizes_near_the_end_of_an_int_are_refused(L, f, bad):
    if f is not lora_q:
        bad = {k: v for k, v in bad.items() if k != "ld_s"}
    assert f(L, **bad, **({} if f is group else dict(ws_bytes=1 << 60))) == ARGS


def test_bytes_that_pass_64_bits_are_refused(L):
    assert L.w2v_lora_workspace_bytes(1 << 60, 3, 128) == -1 and L.w2v_lora_workspace_bytes(10, HUGE, 128) == -1
    per = L.w2v_ctc_beam_state_bytes(1, 32, 128, 16000000)
    n = 0x7fffffff
    assert per > 0 and per * n > (1 << 63) - 1               # (a product of 64 bits would be another number)
    assert L.w2v_ctc_beam_state_bytes(n, 32, 128, 16000000) == -1
    assert beam(L, n_utt=n, width=128, max_frames=16000000, state_bytes=(1 << 63) - 1) == ARGS


@pytest.mark.parametrize("f", [lora, lora_q])
def test_a_workspace_size_is_given_for_what_the_calls_take(L, f):
    """Single rows by the million: up to M + 256 (1 + min(n_utt, M)) = 2^31 - 1 there is a size and the
    calls want that much; past it there is none and they are refused."""
    for rows in (8000000, 8355966):            # 257 rows + 256 <= 2^31 - 1
        need = L.w2v_lora_workspace_bytes(rows, rows, 8)
        assert need > 0 and f(L, M=rows, n_utt=rows, rank=8, ws_bytes=need - 1) == CAPACITY
    for rows in (8355967, 9000000, 100000000):
        assert L.w2v_lora_workspace_bytes(rows, rows, 8) == -1
        assert f(L, M=rows, n_utt=rows, rank=8, ws_bytes=1 << 60) == ARGS
    assert L.w2v_lora_workspace_bytes(2000000000, 3, 8) > 0
