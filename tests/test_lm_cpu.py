"""The decoder's serving step without a GPU: the oracle's own arithmetic, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest

from gpreempt_b200 import binding as B
from gpreempt_b200 import build as gpx_build
from oracle import lm


@pytest.fixture(scope="module")
def lib():
    gpx_build.build()
    return B.load()


def test_codes_round_to_nearest_even():
    torch = pytest.importorskip("torch")
    x = np.concatenate([lm.E4M3[:127], (lm.E4M3[1:127] + lm.E4M3[:126]) / 2, np.random.default_rng(1).standard_normal(4096) * 100])
    x = x[np.abs(x) <= 448].astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(lm.encode(x), want)
    assert np.array_equal(lm.decode(want), torch.from_numpy(want).view(torch.float8_e4m3fn).double().numpy())


def test_block_scales_are_the_smallest_powers_of_two():
    for amax in (448.0, 448.0001, 447.9, 1.0, 1.75, 1.7500001, 3e38, 1e-30, 1e-44):
        x = np.zeros((1, 1, 4), np.float32)
        x[0, 0, 2] = -amax
        scale = float(lm.block_scale(x)[0])
        amax = float(np.float32(amax))
        assert amax <= 448.0 * scale and np.log2(scale) == round(np.log2(scale))
        assert scale == 2.0 ** -126 or amax > 448.0 * scale / 2


def test_cache_refusals(lib):
    h, p = ctypes.c_void_p(), ctypes.c_void_p(1 << 20)

    def make(k=p, v=p, ks=p, vs=p, pages=4, page=64, heads=2, dim=128):
        return lib.gpx_kv_cache_create(k, v, ks, vs, pages, page, heads, dim, ctypes.byref(h))

    assert make(k=None) == B.FAIL and b"NULL" in lib.gpx_last_error()
    assert make(page=48) == B.OUT_OF_RANGE and b"page_tokens" in lib.gpx_last_error()
    assert make(dim=96) == B.OUT_OF_RANGE and b"head_dim" in lib.gpx_last_error()
    assert make(pages=0) == B.OUT_OF_RANGE
    assert make(heads=0) == B.OUT_OF_RANGE
    assert make(pages=1 << 30, page=128, heads=8) == B.OUT_OF_RANGE and b"rows" in lib.gpx_last_error()
    assert make(k=ctypes.c_void_p((1 << 20) + 8)) == B.FAIL and b"aligned" in lib.gpx_last_error()
    assert not h.value
    assert lib.gpx_kv_cache_destroy(None) == B.SUCC


def test_context_size_and_null_arguments(lib):
    n = ctypes.c_size_t()
    assert lib.gpx_lm_ctx_bytes(ctypes.byref(n)) == B.SUCC and n.value > 1 << 20
    assert lib.gpx_lm_ctx_bytes(None) == B.FAIL
    assert lib.gpx_lm_ctx_reset(None, None) == B.FAIL
    assert lib.gpx_lm_status(None, None, None) == B.FAIL
    assert lib.gpx_kv_append(None, None, None, None, None, None) == B.FAIL
    assert lib.gpx_kv_attend(None, None, None, None, None, None) == B.FAIL
    assert lib.gpx_token_scores(None, None, None, None) == B.FAIL


def test_score_refusals(lib):
    ctx, p = ctypes.c_void_p(1 << 20), 1 << 20

    def call(ctx=ctx, **kw):
        a = B.TokenScoresArgs(logits=p, rows=2, vocab=100, inv_temperature=1.0, dtype=b"float32")
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gpx_token_scores(ctypes.byref(a), ctx, None, None)

    assert call(dtype=b"float64") == B.OUT_OF_RANGE and b"float64" in lib.gpx_last_error()
    assert call(dtype=None) == B.FAIL
    assert call(vocab=0) == B.OUT_OF_RANGE
    assert call(rows=-1) == B.OUT_OF_RANGE
    assert call(top=33) == B.OUT_OF_RANGE and b"top" in lib.gpx_last_error()
    assert call(top=9, vocab=8) == B.OUT_OF_RANGE
    assert call(top_ids=p) == B.OUT_OF_RANGE
    assert call(logprob=p) == B.FAIL and b"targets" in lib.gpx_last_error()
    for t in (0.0, -1.0, float("nan"), float("inf")):
        assert call(inv_temperature=t) == B.OUT_OF_RANGE
    assert call(ld=99) == B.OUT_OF_RANGE
    assert call(ctx=ctypes.c_void_p((1 << 20) + 64)) == B.FAIL and b"256" in lib.gpx_last_error()
    word = B.Blp(preempted=p)
    a = B.TokenScoresArgs(logits=p, rows=2, vocab=100, inv_temperature=1.0, dtype=b"float32")
    assert lib.gpx_token_scores(ctypes.byref(a), ctx, ctypes.byref(word), None) == B.FAIL and b"stop_index" in lib.gpx_last_error()


def test_packed_arguments_have_the_structures_layout():
    from gpreempt_b200 import api

    for packed, structure in ((api._APPEND_ARGS, B.KvAppendArgs), (api._ATTEND_ARGS, B.KvAttendArgs), (api._SCORES_ARGS, B.TokenScoresArgs)):
        assert packed.size == ctypes.sizeof(structure)
        values = tuple(range(1, 1 + len(structure._fields_)))
        raw = structure.from_buffer_copy(packed.pack(*values))
        for value, (name, kind) in zip(values, structure._fields_):
            if kind is ctypes.c_char_p:  # (an address that is not to be followed)
                at = getattr(structure, name).offset
                assert int.from_bytes(bytes(raw)[at:at + 8], "little") == value
            else:
                assert getattr(raw, name) == value
