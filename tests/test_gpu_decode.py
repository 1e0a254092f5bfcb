"""The example decoder: its steps against one pass over whole texts, against the oracle, and under interruptions."""
import threading
import time

import numpy as np
import pytest

from oracle import lm

pytestmark = pytest.mark.gpu


def _bits(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


@pytest.mark.parametrize("window", [0, 20])
def test_token_by_token_scores_as_a_whole_text(gpx, window):
    from gpreempt_b200.decode import Decoder

    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, Decoder.VOCAB, n) for n in (70, 1, 33)]
    d = Decoder(3, 110, window=window)
    _, _, tokens = d.step(prompts)
    texts = [list(p) for p in prompts]
    entropies = [[] for _ in prompts]
    for _ in range(30):
        for t, x in zip(texts, tokens):
            t.append(int(x))
        _, entropy, tokens = d.step([[x] for x in tokens])
        for e, x in zip(entropies, entropy):
            e.append(float(x[0]))
    d.status()
    d.free()
    whole = Decoder(3, 110, window=window)
    logprob, entropy, last = whole.step(texts)
    whole.status()
    # rows of the projections are the same bits either way; pages' scales and the order of sums are not, so that attention
    # differs by a rounding to bf16 (2^-8 of it), and the logits by as much of their size (about 8) and a rounding of their own
    allowed = 3 * 8 * 2.0 ** -8
    for s, p in enumerate(prompts):
        assert np.max(np.abs(entropy[s][len(p):] - np.array(entropies[s]))) <= allowed
        # the token chosen at each step is the likeliest one, or ties with it
        chosen = logprob[s][len(p) - 1:]
        assert np.all(np.isfinite(chosen)) and np.all(chosen <= 0)
    # the scores of the first text are those of its restatement
    ids = np.array(texts[0])
    x = _bits(whole.embedding[ids]).astype(np.float64)
    h, kv, dim = whole.HEADS * whole.DIM, whole.KV_HEADS, whole.DIM
    weights = [_bits(w.download(np.uint16).reshape(-1, h)).astype(np.float64) for w in (whole.w_qkv, whole.w_out, whole.w_head)]

    def rounded(y):
        u = y.astype(np.float32).view(np.uint32)
        return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32).astype(np.float64)

    qkv = rounded(x @ weights[0].T).reshape(len(ids), -1, dim)
    n, page = len(ids), whole.PAGE
    cos, sin = whole.cos.download(np.float32).reshape(-1, dim // 2), whole.sin.download(np.float32).reshape(-1, dim // 2)
    pages = -(-n // page)
    k, v = (np.zeros((pages, kv, page, dim), np.uint8) for _ in range(2))
    ks, vs = (np.ones((pages, kv), np.float32) for _ in range(2))
    table = np.arange(pages)[None]
    lm.append(k, v, ks, vs, table, [n], [0, n], qkv[:, whole.HEADS:whole.HEADS + kv], qkv[:, whole.HEADS + kv:], cos, sin, dim, False)
    q = rounded(lm.turn(qkv[:, :whole.HEADS], np.arange(n), cos, sin, dim, False))
    out, _, _ = lm.attend(q, k, v, ks, vs, table, [n], [0, n], window=window)
    logits = rounded(rounded(rounded(out.reshape(n, h)) @ weights[1].T) @ weights[2].T).astype(np.float32)
    want, want_entropy, _, order, _ = lm.scores(logits, np.append(ids[1:], -1).astype(np.int32), 1)
    assert np.max(np.abs(entropy[0] - want_entropy)) <= allowed
    assert np.max(np.abs(logprob[0] - want[:-1])) <= allowed
    whole.free()


def test_a_best_effort_decoder_gives_the_same_tokens_under_interruptions(gpx):
    from gpreempt_b200.decode import Decoder

    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, Decoder.VOCAB, n) for n in (200, 150, 7, 64)]

    def run(word):
        d = Decoder(4, 240, word=word)
        logprob, _, tokens = d.step(prompts)
        out = [np.concatenate(logprob), tokens]
        for _ in range(12):
            _, entropy, tokens = d.step([[t] for t in tokens])
            out += [np.concatenate(entropy), tokens]
        d.status()
        stops = d.stops
        d.free()
        return out, stops

    word = gpx.PreemptWord()
    want, stops = run(word)
    assert stops == 0
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
        got, stops = run(word)
    finally:
        done.set()
        t.join()
        word.clear()
    assert stops > 0
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    word.destroy()
