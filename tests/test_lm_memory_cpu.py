"""Serving in bounded memory without a GPU: the restatement's own arithmetic, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest

from gpreempt_b200 import binding as B
from gpreempt_b200 import build as gpx_build
from oracle import lm

P = 1 << 20  # an address that is never followed


@pytest.fixture(scope="module")
def lib():
    gpx_build.build()
    return B.load()


@pytest.fixture
def cache(lib):
    """What a cache's handle points to (making one needs a driver): codes, scales, pages, page_tokens, kv_heads, dim."""
    def make(kv_heads=2, dim=64, page=16):
        raw = (ctypes.c_uint64 * 64)(P, P, P, P)
        ints = ctypes.cast(ctypes.addressof(raw) + 32, ctypes.POINTER(ctypes.c_int))
        for i, v in enumerate((4, page, kv_heads, dim)):
            ints[i] = v
        return raw
    return make


def batch(seqs=2, tokens=2, most_new=1, table_ld=4, table=P, context=P, first=P):
    return B.KvBatch(table, context, first, table_ld, seqs, tokens, most_new)


def account(**kw):
    a = dict(weights=P, slots=P, ld=100, rows=8, kv_heads=2)
    a.update(kw)
    return B.KvWeights(**a)


def refused(lib, status, text, got):
    assert got == status and text.encode() in lib.gpx_last_error(), (got, lib.gpx_last_error())


def test_append_at_refusals(lib, cache):
    def call(where=True, c=None, ctx=P, b=None, axis=(0,) * 32, **kw):
        a = dict(q=None, k=P, v=P, q_out=None, cos=P, sin=P, heads=4, rotated=64, positions=10, dtype=b"bfloat16")
        w = dict(at=P, axes=2, ld=0)
        for k, v in kw.items():
            (w if k in w else a)[k] = v
        axis = np.array(axis, np.uint8)
        positions = B.KvPositions(w["at"], axis.ctypes.data, w["ld"], w["axes"])
        return lib.gpx_kv_append_at(c or cache(), ctypes.byref(b or batch()), ctypes.byref(B.KvAppendArgs(**a)), ctypes.byref(positions) if where else None,
                                    ctypes.c_void_p(ctx), None, None)

    refused(lib, B.FAIL, "positions", call(where=False))
    refused(lib, B.FAIL, "positions", call(at=None))
    refused(lib, B.FAIL, "positions", call(at=P + 2))
    refused(lib, B.OUT_OF_RANGE, "axes", call(axes=0))
    refused(lib, B.OUT_OF_RANGE, "axes", call(axes=5))
    refused(lib, B.OUT_OF_RANGE, "rotated", call(rotated=12))
    refused(lib, B.FAIL, "tables", call(cos=None))
    refused(lib, B.OUT_OF_RANGE, "multiple of the cache's", call(heads=3))
    refused(lib, B.FAIL, "256", call(ctx=P + 16))
    assert lib.gpx_kv_append_at(None, None, None, None, None, None, None) == B.FAIL


def test_weigh_refusals(lib, cache):
    def call(c=None, b=None, acc=None, ctx=P, **kw):
        a = dict(q=P, lse=P, heads=4, causal=1, scale=0.0, decay=1.0, dtype=b"float16")
        a.update(kw)
        return lib.gpx_kv_weigh(c or cache(), ctypes.byref(b or batch()), ctypes.byref(acc or account()), ctypes.byref(B.KvWeighArgs(**a)), ctypes.c_void_p(ctx),
                                None, None)

    refused(lib, B.FAIL, "NULL", call(q=None))
    refused(lib, B.FAIL, "NULL", call(lse=None))
    refused(lib, B.FAIL, "NULL", call(acc=account(weights=None)))
    refused(lib, B.FAIL, "4-byte", call(acc=account(weights=P + 2)))
    refused(lib, B.FAIL, "4-byte", call(acc=account(slots=P + 1)))
    for kw in (dict(rows=0), dict(ld=0), dict(kv_heads=0), dict(ld=-5)):
        refused(lib, B.OUT_OF_RANGE, "accounts", call(acc=account(**kw)))
    refused(lib, B.OUT_OF_RANGE, "2^60", call(acc=account(ld=1 << 61)))
    refused(lib, B.OUT_OF_RANGE, "rows in accounts", call(acc=account(slots=None, rows=1)))
    refused(lib, B.OUT_OF_RANGE, "for a cache of 2", call(acc=account(kv_heads=4)))
    refused(lib, B.OUT_OF_RANGE, "float32", call(dtype=b"float32"))
    refused(lib, B.OUT_OF_RANGE, "multiple of the cache's", call(heads=5))
    refused(lib, B.OUT_OF_RANGE, "window", call(window=-1))
    refused(lib, B.OUT_OF_RANGE, "window", call(window=2, causal=0))
    refused(lib, B.OUT_OF_RANGE, "observed", call(observed=-1))
    for scale in (-1.0, float("nan"), float("inf")):
        refused(lib, B.OUT_OF_RANGE, "scale", call(scale=scale))
    for decay in (0.0, -1.0, 1.5, float("nan")):
        refused(lib, B.OUT_OF_RANGE, "decay", call(decay=decay))
    refused(lib, B.OUT_OF_RANGE, "longer", call(q_ld=8))
    refused(lib, B.FAIL, "aligned", call(q=P + 8))
    refused(lib, B.FAIL, "aligned", call(q_ld=4 * 64 + 4))
    refused(lib, B.FAIL, "256", call(ctx=P + 64))
    refused(lib, B.OUT_OF_RANGE, "sequences", call(b=batch(seqs=0)))
    word = B.Blp(preempted=P)
    a = B.KvWeighArgs(q=P, lse=P, heads=4, causal=1, decay=1.0, dtype=b"float16")
    refused(lib, B.FAIL, "stop_index", lib.gpx_kv_weigh(cache(), ctypes.byref(batch()), ctypes.byref(account()), ctypes.byref(a), ctypes.c_void_p(P),
                                                        ctypes.byref(word), None))
    assert lib.gpx_kv_weigh(None, None, None, None, None, None, None) == B.FAIL


def test_choose_refusals(lib):
    def call(b=None, acc=None, ctx=P, **kw):
        a = dict(kept=P, counts=P, kept_ld=0, keep=10, first=2, last=3)
        a.update(kw)
        return lib.gpx_kv_choose(ctypes.byref(b or batch()), ctypes.byref(acc or account()), ctypes.byref(B.KvChooseArgs(**a)), ctypes.c_void_p(ctx), None, None)

    refused(lib, B.FAIL, "kept", call(kept=None))
    refused(lib, B.FAIL, "kept", call(counts=P + 2))
    for kw in (dict(keep=0), dict(first=-1), dict(last=-1), dict(first=8), dict(first=2 ** 31 - 1, last=2 ** 31 - 1)):
        refused(lib, B.OUT_OF_RANGE, "keep", call(**kw))
    for ld in (9, -1, 2 ** 31 + 1, 2 ** 63 - 1):
        refused(lib, B.OUT_OF_RANGE, "keeps 10", call(kept_ld=ld))
    refused(lib, B.OUT_OF_RANGE, "heads", call(acc=account(kv_heads=2 ** 31 - 1, ld=1)))
    refused(lib, B.FAIL, "NULL", call(b=batch(context=None)))
    refused(lib, B.FAIL, "256", call(ctx=P + 4))
    assert lib.gpx_kv_choose(None, None, None, None, None, None) == B.FAIL


def test_move_refusals(lib, cache):
    def call(b=None, source=None, to=None, acc=True, to_acc=True, ctx=P, **kw):
        a = dict(to_table=P, kept=P, counts=P, kept_ld=10, to_ld=1)
        a.update(kw)
        acc = account() if acc is True else acc
        to_acc = account(weights=2 * P) if to_acc is True else to_acc
        return lib.gpx_kv_move(source or cache(), ctypes.byref(b or batch()), to or cache(page=32), ctypes.byref(B.KvMoveArgs(**a)),
                               ctypes.byref(acc) if acc else None, ctypes.byref(to_acc) if to_acc else None, ctypes.c_void_p(ctx), None, None)

    refused(lib, B.OUT_OF_RANGE, "caches", call(to=cache(kv_heads=3)))
    refused(lib, B.OUT_OF_RANGE, "caches", call(to=cache(dim=128)))
    for kw in (dict(to_table=None), dict(kept=None), dict(counts=None), dict(kept=P + 2)):
        refused(lib, B.FAIL, "4-byte", call(**kw))
    refused(lib, B.OUT_OF_RANGE, "to_ld", call(to_ld=0))
    for ld in (0, -1, 2 ** 31 + 1, 2 ** 63 - 1):
        refused(lib, B.OUT_OF_RANGE, "kept_ld", call(kept_ld=ld))
    refused(lib, B.FAIL, "one of the accounts", call(acc=None))
    refused(lib, B.FAIL, "one of the accounts", call(to_acc=None))
    refused(lib, B.FAIL, "in place", call(to_acc=account()))
    refused(lib, B.OUT_OF_RANGE, "for a cache of 2", call(to_acc=account(weights=2 * P, kv_heads=1)))
    refused(lib, B.FAIL, "256", call(ctx=P + 4))
    assert lib.gpx_kv_move(None, None, None, None, None, None, None, None, None) == B.FAIL


def test_w4_refusals(lib):
    n = ctypes.c_size_t()

    def w(**kw):
        a = dict(packed=P, n=40, k=256, group=64, zeros=1, dtype=b"float16")
        a.update(kw)
        return B.W4(**a)

    assert lib.gpx_w4_bytes(ctypes.byref(w()), ctypes.byref(n)) == B.SUCC and n.value >= 48 * 128
    for kw in (dict(group=16), dict(group=0), dict(n=0), dict(k=0), dict(k=96), dict(dtype=b"float32")):
        assert lib.gpx_w4_bytes(ctypes.byref(w(**kw)), ctypes.byref(n)) == B.OUT_OF_RANGE
    assert lib.gpx_w4_bytes(None, ctypes.byref(n)) == B.FAIL and lib.gpx_w4_bytes(ctypes.byref(w()), None) == B.FAIL
    pack = lambda weights, c=P, s=P, z=P: lib.gpx_w4_pack(ctypes.byref(weights), c, s, z, None)  # noqa: E731
    refused(lib, B.FAIL, "packed", pack(w(packed=None)))
    refused(lib, B.FAIL, "packed", pack(w(packed=P + 128)))
    refused(lib, B.FAIL, "codes or scales", pack(w(), c=P + 2))
    refused(lib, B.FAIL, "codes or scales", pack(w(), s=None))
    refused(lib, B.FAIL, "zeros", pack(w(), z=None))
    refused(lib, B.FAIL, "zeros", pack(w(zeros=0)))

    def call(weights=None, ctx=P, **kw):
        a = dict(x=P, y=P, rows=3)
        a.update(kw)
        return lib.gpx_w4_matvec(ctypes.byref(weights or w()), ctypes.byref(B.W4MatvecArgs(**a)), ctypes.c_void_p(ctx), None, None)

    refused(lib, B.FAIL, "NULL", call(x=None))
    refused(lib, B.FAIL, "NULL", call(y=None))
    for rows in (0, -1, 65):
        refused(lib, B.OUT_OF_RANGE, "rows", call(rows=rows))
    refused(lib, B.OUT_OF_RANGE, "longer", call(x_ld=128))
    refused(lib, B.OUT_OF_RANGE, "longer", call(y_ld=8))
    refused(lib, B.FAIL, "aligned", call(x=P + 8))
    refused(lib, B.FAIL, "aligned", call(x_ld=260))
    refused(lib, B.FAIL, "256", call(ctx=P + 8))
    assert lib.gpx_w4_matvec(None, None, None, None, None) == B.FAIL


def test_packed_arguments_have_the_structures_layout():
    from gpreempt_b200 import api

    for packed, structure in ((api._WEIGH_ARGS, B.KvWeighArgs), (api._CHOOSE_ARGS, B.KvChooseArgs), (api._MOVE_ARGS, B.KvMoveArgs),
                              (api._MATVEC_ARGS, B.W4MatvecArgs)):
        assert packed.size == ctypes.sizeof(structure)
        raw = packed.pack(*range(1, 1 + len(structure._fields_)))
        for value, (name, kind) in zip(range(1, 100), structure._fields_):
            at = getattr(structure, name)
            if kind is ctypes.c_char_p:
                assert int.from_bytes(raw[at.offset:at.offset + 8], "little") == value
            else:
                assert getattr(structure.from_buffer_copy(raw), name) == value


@pytest.mark.parametrize("zeros", [True, False])
def test_quantised_weights_are_within_half_a_step(zeros):
    from gpreempt_b200 import api

    w = np.random.default_rng(1).standard_normal((5, 256)).astype(np.float32)
    w[2] = np.abs(w[2])
    w[3, :64] = 0
    codes, scales, zero = api.quantize_w4(w, 64, zeros)
    back = lm.w4_weights(codes, scales, zero, 64)
    # a zero is rounded too where a group has one: what it moves is at most half a step at the ends
    assert np.all(np.abs(back - w) <= (1.001 if zeros else 0.501) * scales.repeat(64, 1))
    assert np.all(back[3, :64] == 0)
    with pytest.raises(ValueError):
        api.quantize_w4(w, 48)


def test_the_restatement_of_choosing_and_moving():
    rng = np.random.default_rng(2)
    w = rng.random((1, 1, 9)).astype(np.float32)
    w[0, 0] = [5, 1, 7, 7, np.nan, 0, 7, 2, 3]
    assert lm.choose(w, [0], [9], 4)[0].tolist() == [[2, 3, 4, 6]]
    assert lm.choose(w, [0], [9], 4, 1, 1)[0].tolist() == [[0, 2, 4, 8]]
    assert lm.choose(w, [0], [3], 4)[0].tolist() == [[0, 1, 2]]
    k = lm.encode(rng.standard_normal((3, 1, 4, 8)) * 100)
    scale = np.array([[1.0], [4.0], [0.25]], np.float32)
    to, to_scale = np.zeros((2, 1, 4, 8), np.uint8), np.zeros((2, 1), np.float32)
    lm.move(k, k, scale, scale, np.array([[2, 0, 1]]), [np.array([[0, 5, 6, 7, 11]])], to, to.copy(), to_scale, to_scale.copy(), np.array([[1, 0]]))
    x = lm.decode(k) * scale[:, :, None, None]
    want = [x[2, 0, 0], x[0, 0, 1], x[0, 0, 2], x[0, 0, 3], x[1, 0, 3]]
    got = lm.decode(to) * to_scale[:, :, None, None]
    got = [got[1, 0, 0], got[1, 0, 1], got[1, 0, 2], got[1, 0, 3], got[0, 0, 0]]
    for a, b in zip(got, want):
        assert np.all(np.abs(a - b) <= np.maximum(np.abs(b) * 2.0 ** -4, 2.0 ** -10 * to_scale.max()))


def test_a_sequence_that_ends_leaves_no_positions_behind():
    from gpreempt_b200.decode import Pages

    p = Pages(8, 16, 2, 64)
    p.grow([20, 5])
    p.grow([1, 0])
    assert p.seen.tolist() == [21, 5]
    p.replace(0, p.take(7), 7)  # an eviction: its next token is still its 22nd
    assert p.context.tolist() == [7, 5] and p.seen.tolist() == [21, 5]
    with pytest.raises(MemoryError):
        p.grow([1, 60])
    assert p.seen.tolist() == [21, 5]
    p.release(0)
    assert p.context.tolist() == [0, 5] and p.seen.tolist() == [0, 5]
    p.grow([3, 1])
    assert p.seen.tolist() == [3, 6] and len(p.free) == 6


@pytest.mark.parametrize("keep,room", [(50, 60), (50, 99), (24, 1), (60, 100)])
def test_a_decoder_without_room_to_grow_to_an_eviction_is_refused(keep, room):
    """Before anything is asked of a GPU."""
    from gpreempt_b200.decode import Decoder

    with pytest.raises(ValueError, match="room"):
        Decoder(1, 200, keep=keep, room=room)


def _held_by(x, dtype):
    """x as the products read scales of this type."""
    if dtype == "float16":
        return x.astype(np.float16).astype(np.float64)
    u = x.astype(np.float32).view(np.uint32).astype(np.int64)
    return (((u + 0x7FFF + (u >> 16 & 1)) >> 16 << 16).astype(np.uint32)).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("zeros", [True, False])
def test_codes_belong_to_the_scales_that_the_products_read(zeros, dtype):
    """Codes that are not the outermost ones are within half a step of the 16-bit scale; a division and a product are rounded to 2^-24 of at
    most fifteen steps each."""
    from gpreempt_b200 import api

    w = np.random.default_rng(3).standard_normal((64, 1024)).astype(np.float32)
    w[1] *= 1e-9 if dtype == "float16" else 1e-38  # scales where the type runs out of numbers
    w[2] = 0
    w[3, :128], w[3, 64] = 0, 1e-45
    with np.errstate(all="raise", under="ignore"):
        codes, scales, zero = api.quantize_w4(w, 128, zeros, dtype=dtype)
    assert scales.dtype == np.float32 and np.array_equal(scales, _held_by(scales, dtype)) and np.all(scales > 0)
    q = np.stack([codes & 15, codes >> 4], 2).reshape(64, 8, 128).astype(np.float64)
    offset = 8.0 if zero is None else zero[:, :, None].astype(np.float64)
    steps = np.abs(w.reshape(64, 8, 128) / scales[:, :, None].astype(np.float64) - (q - offset))
    inner = (q > 0) & (q < 15)
    assert np.max(steps[inner]) <= 0.5 + 30 * 2.0 ** -24 and np.max(steps) <= 0.51 + 0.5 * zeros
    back = lm.w4_weights(codes, scales, zero, 128)
    assert np.all(back[2] == 0)


def test_weights_without_a_scale_are_refused():
    from gpreempt_b200 import api

    for value, dtype in ((np.nan, "bfloat16"), (np.inf, "float16"), (1e7, "float16")):
        w = np.ones((2, 64), np.float32)
        w[1, 5] = value
        with pytest.raises(ValueError, match="scale"):
            api.quantize_w4(w, 32, dtype=dtype)
    with pytest.raises(ValueError, match="float32"):
        api.quantize_w4(np.ones((2, 64)), 32, dtype="float32")


def test_weights_that_are_gone_have_no_address(lib):
    """Products with them are refused, not run over memory that may be anybody's."""
    from gpreempt_b200 import api

    w = api.FourBit.__new__(api.FourBit)
    w.struct = B.W4(P, 16, 64, 64, 1, b"bfloat16")
    w._ref, w._buf = ctypes.byref(w.struct), api.DeviceBuffer.__new__(api.DeviceBuffer)
    w._buf.ptr = ctypes.c_void_p()  # (no device memory here)
    w.free()
    assert w.struct.packed is None
    a = B.W4MatvecArgs(x=P, y=P, rows=1)
    refused(lib, B.FAIL, "packed", lib.gpx_w4_matvec(w._ref, ctypes.byref(a), ctypes.c_void_p(P), None, None))
