"""Serving in bounded memory, stopped where work is under way: launches that have run tiles and have some left, tiles of accounts that stop
between two chunks of rows, rows of products whose parts were brought by different launches.  A stop counts here only if the launch had begun."""
import time

import numpy as np
import pytest

from test_gpu_lm import Bed, tables, to_bits
from test_gpu_lm_memory import Account, Moved, free, up, weights_of

pytestmark = pytest.mark.gpu

COUNTERS, HEADER, NOTES = 65536, 256, 1024  # of a context: ints behind its header, the last ones are what unfinished tiles note


@pytest.fixture(scope="module")
def ctx(gpx):
    c = gpx.LmContext()
    yield c
    assert c.status() == (0, 0)
    c.free()


def notes(ctx):
    return ctx.buf.download(np.int32, NOTES, offset=HEADER + 4 * (COUNTERS - NOTES))


def joins(ctx):
    return ctx.buf.download(np.int32, COUNTERS - NOTES, offset=HEADER)


def stopped_runs(gpx, ctx, launch, read, fresh, run_us, under_way=lambda ctx: True, enough=3, trials=60, clean=True):
    """Raises the word at various moments of a launch and of the one that goes on with it, until `enough` launches have stopped with tiles
    behind them and `under_way` has found what they left; each time all of it must come to the bits of a launch that nobody stopped."""
    word = gpx.PreemptWord(1)
    blp, s = gpx.BlpContext(word, kernel_id=5), gpx.Stream(1)
    fresh()
    launch(blp, s)
    s.sync()
    assert blp.read()["stop_index"] == -1
    want, found = read(), 0
    for trial in range(trials):
        fresh()
        blp.reset()
        gpx.device_sync()
        run = 0
        for rounds in range(30):
            launch(blp, s)
            if rounds < 2:
                t0 = time.perf_counter()
                while (time.perf_counter() - t0) * 1e6 < run_us * (1 + trial % 10) / 11:
                    pass
                word.raise_()
            s.sync()
            word.clear()
            gpx.device_sync()
            st = blp.read()
            if st["stop_index"] == -1:
                break
            assert st["stop_index"] == 5
            found += st["tiles_run"] > run and under_way(ctx)
            run = st["tiles_run"]
            blp.rearm()
        else:
            raise AssertionError("not complete after 30 launches")
        for a, b in zip(read(), want):
            assert np.array_equal(a, b)
        assert not clean or not (notes(ctx).any() or joins(ctx).any())  # nothing is left behind
        if found >= enough:
            break
    assert found >= enough, found
    for o in (blp, word, s):
        (o.free if hasattr(o, "free") else o.destroy)()
    return want


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("window", [0, 5000])
def test_a_tile_of_accounts_stops_between_two_chunks(gpx, ctx, dtype, window):
    """Fewer tiles than CTAs, each of hundreds of chunks: whatever stops, stops in the middle of tiles.  (tiles_run counts the rounds of a CTA.)"""
    new, context, heads, kv, dim, page = [5000], [19000], 16, 1, 128, 64
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=4).upload()
    dq = up(gpx, to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype))
    out, lse = gpx.DeviceBuffer(dq.nbytes), gpx.DeviceBuffer(bed.tokens * heads * 4)
    gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, dtype, ctx, window=window, lse=lse)
    gpx.device_sync()
    account = Account(gpx, bed)

    def stopped(ctx):
        n = notes(ctx)
        assert np.all(n[0::2] <= kv * -(-context[0] // 128))
        return np.count_nonzero(n[0::2]) > 0

    want = stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_weigh(bed.cache, bed.batch, dq, lse, account.handle, heads, dtype, ctx, window=window, decay=0.9,
                                                              blp=blp, stream=s),
                        lambda: [account.read()], lambda: account.dw.upload(account.w), 600, stopped)
    account.dw.upload(account.w)
    gpx.kv_weigh(bed.cache, bed.batch, dq, lse, account.handle, heads, dtype, ctx, window=window, decay=0.9)
    gpx.device_sync()
    assert np.array_equal(account.read(), want[0])
    free(dq, out, lse, account, bed)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_accounts_behind_attention_that_was_stopped(gpx, dtype):
    """Attention of a prompt stops in the middle of tiles and is resumed; preemptible accounts of the same prompt in the same context then have
    nothing to go on with."""
    new, context, heads, kv, dim, page = [3000, 900], [19000, 900], 16, 4, 128, 64
    mine, other = gpx.LmContext(), gpx.LmContext()
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=4).upload()
    dq = up(gpx, to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype))
    out, lse = gpx.DeviceBuffer(dq.nbytes), gpx.DeviceBuffer(bed.tokens * heads * 4)
    stopped_runs(gpx, mine, lambda blp, s: gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, dtype, mine, lse=lse, blp=blp, stream=s),
                 lambda: [out.download(np.uint16), lse.download(np.float32)], out.zero, 800, lambda ctx: notes(ctx)[2::4].any(), clean=False)
    account = Account(gpx, bed)
    word, got = gpx.PreemptWord(), []
    for ctx in (other, mine):
        blp = gpx.BlpContext(word)
        account.dw.upload(account.w)
        gpx.kv_weigh(bed.cache, bed.batch, dq, lse, account.handle, heads, dtype, ctx, decay=0.5, blp=blp)
        gpx.device_sync()
        assert blp.read()["stop_index"] == -1 and ctx.status() == (0, 0)
        got.append(account.read())
        blp.free()
    assert np.array_equal(*got)
    assert not notes(mine).any() and not joins(mine).any()
    word.destroy()
    free(mine, other, dq, out, lse, account, bed)


@pytest.mark.parametrize("rows,group,zeros", [(1, 64, False), (24, 32, True), (64, 128, True)])
def test_rows_of_products_whose_parts_two_launches_bring(gpx, ctx, rows, group, zeros):
    n, k = 30011, 16384
    rng = np.random.default_rng(1)
    codes, scales = up(gpx, rng.integers(0, 256, (n, k // 2), np.uint8)), up(gpx, to_bits(rng.random((n, k // group)) * 0.02, "bfloat16"))
    z = up(gpx, rng.integers(0, 16, (n, k // group)).astype(np.uint8)) if zeros else None
    w = gpx.FourBit(codes, scales, z, n, k, group, "bfloat16")
    x, y = up(gpx, to_bits(rng.standard_normal((rows, k)), "bfloat16")), gpx.DeviceBuffer(rows * n * 2)
    stopped_runs(gpx, ctx, lambda blp, s: gpx.w4_matvec(w, x, y, rows, ctx, blp=blp, stream=s), lambda: [y.download(np.uint16)], y.zero,
                 100 if rows == 1 else 200, lambda ctx: joins(ctx).any())
    free(codes, scales, w, x, y, *([z] if zeros else []))


@pytest.mark.parametrize("new,seqs,context", [(1, 40, 10000), (12, 20, 20000)])
def test_accounts_of_few_rows_stop_between_tiles(gpx, ctx, new, seqs, context):
    heads, kv, dim, page = 16, 4, 128, 64
    bed = Bed(gpx, [new] * seqs, [context - 31 * i for i in range(seqs)], heads, kv, dim, page, seed=4).upload()
    dq, lse = up(gpx, to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), "bfloat16")), up(gpx, np.full((bed.tokens, heads), 9, np.float32))
    account = Account(gpx, bed)
    stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_weigh(bed.cache, bed.batch, dq, lse, account.handle, heads, "bfloat16", ctx, decay=0.9, blp=blp, stream=s),
                 lambda: [account.read()], lambda: account.dw.upload(account.w), 80)
    free(dq, lse, account, bed)


@pytest.mark.parametrize("kind", ["spread", "ties"])
@pytest.mark.parametrize("seqs,most", [(100, 20000), (14, 60000)])
def test_choosing_stops_between_tiles(gpx, ctx, kind, seqs, most):
    """Accounts that are read in pieces, more of them than are looked at at once; and few with 1 024 threads each, of which all have begun
    before a stop can be seen."""
    kv, keep = 8, 4000
    context = np.array([most - 30 * i for i in range(seqs)], np.int32)
    w = up(gpx, weights_of(kind, (seqs, kv, most), np.random.default_rng(2)))
    arrays = [up(gpx, a) for a in (np.zeros((seqs, 1), np.int32), context, np.zeros(seqs + 1, np.int32))]
    batch, account = gpx.KvBatch(seqs, 0, 0, *arrays, 1), gpx.KvWeights(w, seqs, kv, most)
    kept, counts = gpx.DeviceBuffer(seqs * kv * keep * 4), gpx.DeviceBuffer(seqs * 4)
    few = seqs * kv <= 148
    stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_choose(batch, account, kept, counts, keep, ctx, 4, 100, blp=blp, stream=s),
                 lambda: [kept.download(np.int32), counts.download(np.int32)], lambda: (kept.zero(), counts.zero()), 10 if few else 120,
                 enough=0 if few else 3, trials=12 if few else 60)
    free(w, kept, counts, *arrays)


def test_moving_stops_between_tiles(gpx, ctx):
    seqs, kv, dim, page, keep = 40, 8, 64, 64, 3000
    bed = Bed(gpx, [0] * seqs, [6000 - 30 * i for i in range(seqs)], kv, kv, dim, page, seed=4).upload()
    lists = np.sort(bed.rng.random((seqs, kv, 4800)).argsort(2)[:, :, :keep].astype(np.int32), 2)
    kept, counts = up(gpx, lists), up(gpx, np.full(seqs, keep, np.int32))
    account, to, to_account = Account(gpx, bed), Moved(gpx, bed, [keep] * seqs, 16), Account(gpx, bed, seed=5)

    def fresh():
        for b, a in zip(to.buffers, (to.k, to.v, to.ks, to.vs)):
            b.upload(a)
        to_account.dw.upload(to_account.w)

    stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_move(bed.cache, bed.batch, to.cache, to.dt, to.table.shape[1], kept, counts, keep, ctx,
                                                      account.handle, to_account.handle, blp=blp, stream=s),
                 lambda: [*to.download(), to_account.read()], fresh, 80)
    free(kept, counts, account, to_account, to, bed)


def test_append_at_stops_between_tiles(gpx, ctx):
    new, heads, kv, dim, page = [6000, 5000, 8000], 8, 8, 128, 64
    context = [n + 77 for n in new]
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=6).upload()
    x = up(gpx, to_bits(bed.rng.standard_normal((bed.tokens, 3 * heads * dim)), "bfloat16"))
    q, width = gpx.DeviceBuffer(bed.tokens * heads * dim * 2), 3 * heads * dim
    cos, sin = tables(4001, dim)
    dcos, dsin, dat = up(gpx, cos), up(gpx, sin), up(gpx, bed.rng.integers(0, 4001, (bed.tokens, 3)).astype(np.int32))
    rope, where = gpx.Rope(dcos, dsin, 4001, dim), gpx.KvPositions(dat, 3, np.arange(dim // 2) % 3)

    def fresh():
        q.zero()
        for b, a in ((bed.dk, bed.k), (bed.dv, bed.v), (bed.dks, bed.ks), (bed.dvs, bed.vs)):
            b.upload(a)

    at = x.ptr.value
    stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_append_at(bed.cache, bed.batch, at, at + 2 * heads * dim, at + 4 * heads * dim, q, heads, "bfloat16",
                                                           ctx, rope, where, blp, s, width, width, width),
                 lambda: [q.download(np.uint16), *bed.download()], fresh, 120)
    free(x, q, dcos, dsin, dat, bed)


@pytest.mark.parametrize("new,most", [(1, 30000), (4, 20000)])
def test_attention_of_few_rows_leaves_nothing_in_the_context(gpx, ctx, new, most):
    heads, kv, dim, page, seqs = 16, 4, 128, 64, 12
    bed = Bed(gpx, [new] * seqs, [most - 501 * i for i in range(seqs)], heads, kv, dim, page, seed=4).upload()
    dq = up(gpx, to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), "bfloat16"))
    out = gpx.DeviceBuffer(dq.nbytes)
    stopped_runs(gpx, ctx, lambda blp, s: gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, "bfloat16", ctx, blp=blp, stream=s),
                 lambda: [out.download(np.uint16)], out.zero, 100)
    free(dq, out, bed)


def test_scores_leave_nothing_in_the_context(gpx, ctx):
    rows, vocab = 4000, 20000
    x = up(gpx, to_bits(np.random.default_rng(1).standard_normal((rows, vocab)) * 4, "float16"))
    entropy, ids = gpx.DeviceBuffer(rows * 4), gpx.DeviceBuffer(rows * 4)
    stopped_runs(gpx, ctx, lambda blp, s: gpx.token_scores(x, rows, vocab, "float16", ctx, None, None, entropy, top=1, top_ids=ids, blp=blp, stream=s),
                 lambda: [entropy.download(np.float32), ids.download(np.int32)], lambda: (entropy.zero(), ids.zero()), 60)
    free(x, entropy, ids)
