"""The example decoder in bounded memory: nothing changes until something is dropped, what is dropped is what weighed least, weights of 4
bits, interruptions."""
import threading
import time

import numpy as np
import pytest

from oracle import lm

pytestmark = pytest.mark.gpu


def _decode(d, prompts, steps):
    logprob, _, tokens = d.step(prompts)
    out = [np.concatenate(logprob), tokens]
    for _ in range(steps):
        _, entropy, tokens = d.step([[t] for t in tokens])
        out += [np.concatenate(entropy), tokens]
    d.status()
    return out


def test_a_decoder_that_drops_nothing_is_the_same(gpx):
    from gpreempt_b200.decode import Decoder

    prompts = [np.random.default_rng(3).integers(0, Decoder.VOCAB, n) for n in (70, 1, 33)]
    results = []
    for keep in (0, 60):
        d = Decoder(3, 110, keep=keep)
        results.append(_decode(d, prompts, 12))
        assert d.evicted == 0
        d.free()
    for a, b in zip(*results):
        assert np.array_equal(a, b)


def test_conversations_keep_what_weighed_most(gpx):
    from gpreempt_b200.decode import Decoder

    keep, room = 24, 60
    rng = np.random.default_rng(4)
    d = Decoder(3, 200, keep=keep, room=room)
    ld, checked = d.account.struct.ld, 0
    evict = d._evict

    def cache():
        c = d.cache
        shape = (c.pages, c.kv_heads, c.page_tokens, c.head_dim)
        return [c.k.download(np.uint8).reshape(shape), c.v.download(np.uint8).reshape(shape), c.k_scale.download(np.float32).reshape(shape[:2]),
                c.v_scale.download(np.float32).reshape(shape[:2])]

    def watched(which):
        nonlocal checked
        d.stream.sync()
        weights, before, table = d.w_now.download(np.float32).reshape(3, d.KV_HEADS, ld), cache(), d.pages.table.copy()
        context = d.pages.context.copy()
        held = [w.copy() for w in weights]
        evict(which)
        d.stream.sync()
        after, now = cache(), d.w_now.download(np.float32).reshape(3, d.KV_HEADS, ld)
        lists = lm.choose(weights, which, context[which], keep, d.FIRST, keep // 4)
        want = [a.copy() for a in before]
        lm.move(*before, table[which], lists, *want, d.pages.table[which])
        for i, some in zip(which, lists):
            n_pages = -(-keep // d.PAGE)
            pages = d.pages.table[i, :n_pages]
            for a, b in zip(after, want):
                assert np.array_equal(a[pages], b[pages])
            for h in range(d.KV_HEADS):
                assert np.array_equal(now[i, h, :keep], held[i][h, some[h]])
            assert d.pages.context[i] == keep
            checked += 1
        # no page is anybody's twice
        used = [int(p) for i in range(3) for p in d.pages.table[i, :-(-int(d.pages.context[i]) // d.PAGE)]]
        assert len(set(used)) == len(used) and not set(used) & set(d.pages.free) and len(used) + len(d.pages.free) == d.cache.pages

    d._evict = watched
    prompts = [rng.integers(0, d.VOCAB, n) for n in (58, 5, 30)]
    out = _decode(d, prompts, 70)
    assert checked == d.evicted >= 5
    assert d.seen.tolist() == [58 + 70, 5 + 70, 30 + 70] and d.pages.context.max() < 2 * keep + 1
    assert all(np.all(np.isfinite(x)) for x in out)
    # a conversation whose positions have run out is refused, and nothing has changed
    seen, context = d.seen.copy(), d.pages.context.copy()
    with pytest.raises(MemoryError):
        d.step([[1] * 30, [1], [1] * 120])
    assert np.array_equal(d.seen, seen) and np.array_equal(d.pages.context, context)
    d.free()


def test_weights_of_four_bits(gpx):
    """Steps of single tokens against the same with those weights as bf16: each differs from its 4-bit one by a rounding (2^-9), a
    product of 512 by less than that of its size, and logits of about 8 by as much and roundings to bf16 on the way."""
    from gpreempt_b200.decode import Decoder, _bf16

    prompts = [np.random.default_rng(6).integers(0, Decoder.VOCAB, n) for n in (3, 1, 2, 1)]
    d = Decoder(4, 40, four_bit=True)
    got = _decode(d, prompts, 1)
    d.free()
    rng = np.random.default_rng(1)
    h = Decoder.HEADS * Decoder.DIM
    rng.standard_normal((Decoder.VOCAB, h))
    plain = Decoder(4, 40)
    for buffer, n, s in ((plain.w_qkv, plain.width, 1.5), (plain.w_out, h, 1.0), (plain.w_head, Decoder.VOCAB, 2.0)):
        codes, scales, zeros = gpx.quantize_w4(rng.standard_normal((n, h)) * s / h ** 0.5, Decoder.GROUP)
        scales = (_bf16(scales).astype(np.uint32) << 16).view(np.float32)
        buffer.upload(_bf16(lm.w4_weights(codes, scales, zeros, Decoder.GROUP)))
    want = _decode(plain, prompts, 1)
    plain.free()
    allowed = 4 * 8 * 2.0 ** -8
    for a, b in zip(got[:1] + got[2:3], want[:1] + want[2:3]):
        if np.array_equal(got[1], want[1]):  # (the same tokens were chosen)
            assert np.max(np.abs(a - b)) <= allowed
    assert np.max(np.abs(got[0] - want[0])) <= allowed


def test_a_best_effort_decoder_in_bounded_memory_under_interruptions(gpx):
    from gpreempt_b200.decode import Decoder

    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, Decoder.VOCAB, n) for n in (100, 90, 7, 64)]

    def run(word):
        d = Decoder(4, 240, word=word, keep=50, room=110, four_bit=True)
        out = _decode(d, prompts, 60)
        stops, evicted = d.stops, d.evicted
        d.free()
        return out, stops, evicted

    word = gpx.PreemptWord()
    want, stops, evicted = run(word)
    assert stops == 0 and evicted >= 4
    done = threading.Event()

    def interrupt():
        while not done.is_set():
            word.raise_()
            time.sleep(0.0002)
            word.clear()
            time.sleep(0.0003)

    t = threading.Thread(target=interrupt)
    t.start()
    try:
        got, stops, _ = run(word)
    finally:
        done.set()
        t.join()
        word.clear()
    assert stops > 0
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    word.destroy()


def test_a_conversation_that_has_ended_leaves_its_place_as_it_was(gpx):
    """After evictions and the end of all conversations the next ones come to the bits of a decoder that has had none."""
    from gpreempt_b200.decode import Decoder

    rng = np.random.default_rng(8)
    before, after = ([rng.integers(0, Decoder.VOCAB, n) for n in lengths] for lengths in ((50, 30, 9), (20, 48, 33)))
    fresh = Decoder(3, 150, keep=24, room=60)
    want = _decode(fresh, after, 60)
    fresh.free()
    d = Decoder(3, 150, keep=24, room=60)
    _decode(d, before, 60)
    assert d.evicted >= 3
    for s in range(3):
        d.pages.release(s)
    got = _decode(d, after, 60)
    assert d.seen.tolist() == [80, 108, 93]
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    d.free()
