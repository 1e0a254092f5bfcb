"""Serving in bounded memory, stopped where work is under way: tiles of accounts that stop between two chunks of rows.  A stop counts here only
if the launch had begun."""
import time

import numpy as np
import pytest

from test_gpu_lm import Bed, to_bits
from test_gpu_lm_memory import Account, free, up

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
