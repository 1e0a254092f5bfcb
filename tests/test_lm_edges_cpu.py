"""What the decoder's serving step refuses on the host, and what its example leaves as it was when it refuses."""
import ctypes

import numpy as np
import pytest

from gpreempt_b200 import binding as B
from gpreempt_b200 import build as gpx_build
from gpreempt_b200.decode import Decoder, Pages


@pytest.fixture(scope="module")
def lib():
    gpx_build.build()
    return B.load()


@pytest.mark.parametrize("name", ["targets", "logprob", "entropy", "lse", "top_ids", "top_logprob"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_scores_refuse_arrays_off_their_boundary(lib, name, off):
    p = 1 << 20
    a = B.TokenScoresArgs(logits=p, targets=p, rows=2, vocab=100, top=3, inv_temperature=1.0, dtype=b"float32")
    setattr(a, name, p + off)
    assert lib.gpx_token_scores(ctypes.byref(a), ctypes.c_void_p(p), None, None) == B.FAIL
    assert b"aligned" in lib.gpx_last_error()


# ---- the example's pages -----------------------------------------------------------------------------

def state_of(p):
    return p.context.tolist(), p.table.tolist(), list(p.free)


@pytest.mark.parametrize("new", [[1, 1, 60], [16, 16, 16], [0, 0, 33], [1, 49, 1]])
def test_a_refused_step_takes_no_pages(new):
    """The sequence at fault comes behind others that would have had their pages."""
    p = Pages(5, 16, 3, 48)
    p.grow([10, 5, 16])
    before = state_of(p)
    with pytest.raises(MemoryError):
        p.grow(new)
    assert state_of(p) == before
    p.release(1)
    assert p.grow([1, 0, 16]).tolist() == [0, 1, 1, 17]
    assert p.context.tolist() == [11, 0, 32]


@pytest.mark.parametrize("most", [50, 1, 16, 47])
def test_a_sequence_ends_at_its_most_tokens_not_at_its_last_page(most):
    """Rotation tables and buffers are made for `most` tokens a sequence; its pages have room for more."""
    p = Pages(100, 32, 2, most)
    p.grow([most - 1, 0])
    before = state_of(p)
    for new in ([2, 0], [1, most + 1]):
        with pytest.raises(MemoryError):
            p.grow(new)
        assert state_of(p) == before
    p.grow([1, most])
    assert p.context.tolist() == [most, most]


@pytest.mark.parametrize("token", [-1, 4096, 1 << 40])
def test_a_step_with_a_token_outside_the_vocabulary_changes_nothing(token):
    d = Decoder.__new__(Decoder)  # (what a step looks at before it asks the device for anything)
    d.seqs, d.pages, d.embedding = 2, Pages(4, 32, 2, 64), np.zeros((Decoder.VOCAB, 8), np.uint16)
    before = state_of(d.pages)
    with pytest.raises(ValueError):
        d.step([[1, 2], [3, token]])
    assert state_of(d.pages) == before
