"""A decoder of one attention layer, served over the paged 8-bit cache: prompts are taken in and scored together, then one
token a conversation and step is chosen, as a latency-critical tenant or as a preemptible best-effort one.

    python -m gpreempt_b200.decode [--conversations 8] [--steps 32] [--best-effort] [--window N]

It shows the operators as they are used together: projections by the framework's GEMM, kv_append with the rotation,
kv_attend, and token_scores for the log probabilities and the choice.  Weights are random.
"""
from __future__ import annotations

import argparse
import time

import numpy as np

from . import api


class Pages:
    """Which pages of a pool hold which sequence: a free list, and a table that grows with the sequences."""

    def __init__(self, pages: int, page_tokens: int, seqs: int, most_tokens: int):
        self.page_tokens, self.most_tokens = page_tokens, most_tokens
        self.free = list(range(pages - 1, -1, -1))
        self.table = np.full((seqs, -(-most_tokens // page_tokens)), -1, np.int32)
        self.context = np.zeros(seqs, np.int32)

    def grow(self, new) -> np.ndarray:
        """Makes room for new[s] tokens of each sequence, or for none of them (MemoryError); returns the offsets of the
        sequences' new tokens."""
        need, left = [], len(self.free)
        for s, n in enumerate(new):
            have, want = (-(-int(c) // self.page_tokens) for c in (self.context[s], self.context[s] + n))
            left -= want - have
            if self.context[s] + n > self.most_tokens:
                raise MemoryError(f"sequence {s} has {self.context[s]} tokens of {self.most_tokens}, {n} more do not fit")
            if left < 0:
                raise MemoryError(f"sequence {s} needs {want - have} more pages")
            need.append(range(have, want))
        for s, n in enumerate(new):
            for i in need[s]:
                self.table[s, i] = self.free.pop()
            self.context[s] += n
        return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)

    def release(self, s: int) -> None:
        used = -(-int(self.context[s]) // self.page_tokens)
        self.free.extend(int(p) for p in self.table[s, :used])
        self.context[s] = 0


def _bf16(x: np.ndarray) -> np.ndarray:
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


class Decoder:
    """Weights, cache and buffers of a tenant; `word` makes its launches preemptible."""

    HEADS, KV_HEADS, DIM, PAGE, VOCAB, TILE = 8, 2, 64, 32, 4096, 128

    def __init__(self, seqs: int, most_tokens: int, seed: int = 1, word: api.PreemptWord | None = None, window: int = 0):
        h, self.seqs, self.most_tokens, self.window = self.HEADS * self.DIM, seqs, most_tokens, window
        rng = np.random.default_rng(seed)
        self.width = (self.HEADS + 2 * self.KV_HEADS) * self.DIM
        upload = api.DeviceBuffer.from_numpy
        self.embedding = _bf16(rng.standard_normal((self.VOCAB, h)))
        self.w_qkv, self.w_out, self.w_head = (
            upload(_bf16(rng.standard_normal((n, h)) * s / h ** 0.5)) for n, s in ((self.width, 1.5), (h, 1.0), (self.VOCAB, 2.0)))
        pages = seqs * -(-most_tokens // self.PAGE)
        self.pages = Pages(pages, self.PAGE, seqs, most_tokens)
        self.cache = api.KvCache(pages, self.PAGE, self.KV_HEADS, self.DIM)
        half = self.DIM // 2
        angle = np.arange(most_tokens)[:, None] * 10000.0 ** (-np.arange(half) / half)
        self.cos, self.sin = upload(np.cos(angle).astype(np.float32)), upload(np.sin(angle).astype(np.float32))
        self.rope = api.Rope(self.cos, self.sin, most_tokens, self.DIM)
        self.stream = api.Stream(0 if word is None else 1)
        self.ctx, self.blp = api.LmContext(), api.BlpContext(word) if word is not None else None
        self.gemm_ctxs = [api.GemmContext() for _ in range(3)]  # (one each: a reset must not meet the product before)
        self.stops = 0
        rows = -(-seqs * most_tokens // self.TILE) * self.TILE
        buffer = api.DeviceBuffer
        self.x, self.qkv, self.q, self.o, self.y, self.logits = (
            buffer(rows * n * 2) for n in (h, self.width, h, h, h, self.VOCAB))
        self.targets, self.logprob, self.entropy, self.best = (buffer(rows * 4) for _ in range(4))
        self.table, self.context, self.first = (buffer(a.nbytes) for a in (self.pages.table, self.pages.context, np.empty(seqs + 1, np.int32)))
        for b in (self.x, self.o):
            b.zero()

    def _run(self, launch) -> None:
        """A launch of a preemptible tenant goes on where it was interrupted until it is complete."""
        if self.blp is None:
            launch()
            return
        self.blp.reset()
        launch()
        self.stream.sync()
        while self.blp.read()["stop_index"] != -1:
            self.stops += 1
            while self.blp.word.value:
                time.sleep(0)
            self.blp.rearm()
            launch()
            self.stream.sync()

    def _gemm(self, which: int, a, b, c, rows: int, n: int) -> None:
        m, ctx = -(-rows // self.TILE) * self.TILE, self.gemm_ctxs[which]
        ctx.reset()
        self._run(lambda: api.gemm_bf16(a, b, c, m, n, self.HEADS * self.DIM, ctx, self.blp, self.stream))

    def step(self, tokens: list) -> tuple:
        """Takes in tokens[s] (arrays, some may be empty) of every sequence.  Returns for each the log probabilities of its
        tokens behind the first, the entropies behind each token, and the most likely next token (-1 without new ones).
        (Prompts and single tokens share a call here; a server with many of both in a step makes one for each.)"""
        new = [len(t) for t in tokens]
        ids = np.concatenate([np.asarray(t, np.int64) for t in tokens])
        if np.any((ids < 0) | (ids >= self.VOCAB)):
            raise ValueError(f"tokens are 0 to {self.VOCAB - 1}")
        first, rows, h = self.pages.grow(new), sum(new), self.HEADS * self.DIM
        if rows == 0:
            return [np.empty(0, np.float32)] * self.seqs, [np.empty(0, np.float32)] * self.seqs, np.full(self.seqs, -1)
        targets = np.full(rows, -1, np.int32)
        for s in range(self.seqs):
            if new[s] > 1:
                targets[first[s]:first[s + 1] - 1] = ids[first[s] + 1:first[s + 1]]
        s, bf = self.stream, "bfloat16"
        for buf, a in ((self.x, self.embedding[ids]), (self.targets, targets), (self.table, self.pages.table), (self.context, self.pages.context),
                       (self.first, first)):
            buf.upload(a, s)
        batch = api.KvBatch(self.seqs, rows, max(new), self.table, self.context, self.first, self.pages.table.shape[1])
        at = self.qkv.ptr.value
        k, v = at + 2 * h, at + 2 * (h + self.KV_HEADS * self.DIM)
        self._gemm(0, self.x, self.w_qkv, self.qkv, rows, self.width)
        self._run(lambda: api.kv_append(self.cache, batch, at, k, v, self.q, self.HEADS, bf, self.ctx, self.rope, self.blp, s, self.width,
                                        self.width, self.width))
        self._run(lambda: api.kv_attend(self.cache, batch, self.q, self.o, self.HEADS, bf, self.ctx, window=self.window, blp=self.blp, stream=s))
        self._gemm(1, self.o, self.w_out, self.y, rows, h)
        self._gemm(2, self.y, self.w_head, self.logits, rows, self.VOCAB)
        self._run(lambda: api.token_scores(self.logits, rows, self.VOCAB, bf, self.ctx, self.targets, self.logprob, self.entropy, top=1,
                                           top_ids=self.best, blp=self.blp, stream=s))
        s.sync()
        logprob, entropy, best = (b.download(t, rows) for b, t in ((self.logprob, np.float32), (self.entropy, np.float32), (self.best, np.int32)))
        span = [slice(first[i], first[i + 1]) for i in range(self.seqs)]
        return ([logprob[r][:-1] for r in span], [entropy[r] for r in span],
                np.array([best[r.stop - 1] if r.stop > r.start else -1 for r in span]))

    def status(self) -> None:
        code, where = self.ctx.status()
        if code or any(c.status()[0] for c in self.gemm_ctxs):
            raise RuntimeError(f"a launch reported {code} at {where}")

    def free(self) -> None:
        self.cache.free()
        for b in (self.w_qkv, self.w_out, self.w_head, self.cos, self.sin, self.x, self.qkv, self.q, self.o, self.y, self.logits, self.targets,
                  self.logprob, self.entropy, self.best, self.table, self.context, self.first, self.ctx, *self.gemm_ctxs):
            b.free()
        if self.blp is not None:
            self.blp.free()
        self.stream.destroy()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--conversations", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=100, help="tokens of the longest prompt")
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--best-effort", action="store_true", help="preemptible launches (nobody raises their word here: what polling costs)")
    a = ap.parse_args()
    api.init_cuda(0)
    word = api.PreemptWord() if a.best_effort else None
    d = Decoder(a.conversations, a.prompt + a.steps, word=word, window=a.window)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, d.VOCAB, max(1, a.prompt - 7 * s % a.prompt)) for s in range(a.conversations)]
    t0 = time.perf_counter()
    logprob, _, tokens = d.step(prompts)
    t1 = time.perf_counter()
    for _ in range(a.steps - 1):
        _, entropy, tokens = d.step([[t] for t in tokens])
    t2 = time.perf_counter()
    d.status()
    scored = np.concatenate(logprob)
    print(f"prompts: {sum(map(len, prompts))} tokens in {(t1 - t0) * 1e3:.2f} ms, mean log probability {scored.mean() if scored.size else 0.0:.3f}")
    if a.steps > 1:
        print(f"{a.steps - 1} steps of {a.conversations} tokens: {(t2 - t1) / (a.steps - 1) * 1e6:.0f} us a step, "
              f"mean entropy of the last {np.mean(np.concatenate(entropy)):.3f}")
    d.free()


if __name__ == "__main__":
    main()
