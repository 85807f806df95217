"""Which beam search the oracle answers with, and that it says so."""
import warnings

import numpy as np
import oracle as O
import pytest


def logits(seed):
    rng = np.random.default_rng(seed)
    lg = rng.standard_normal((40, 12)).astype(np.float32)
    lg[:, 0] += 2.0
    return lg


def test_without_the_reference_it_warns(monkeypatch, tmp_path):
    """The restatement, with a warning."""
    monkeypatch.setattr(O, "REF_LIB", tmp_path / "none.so")
    with pytest.warns(UserWarning, match="restatement"):
        got = O.ref_beam_search(logits(1), 0, 6)
    assert got == O._table_beam_search(logits(1), 0, 6)


@pytest.mark.skipif(not O.ref_available(), reason="no build of the reference")
def test_with_the_reference_it_agrees_and_is_silent():
    for seed in range(6):
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            ref = O.ref_beam_search(logits(seed), 0, 6)
        assert O._table_beam_search(logits(seed), 0, 6) == ref
