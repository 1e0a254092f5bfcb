"""Serving in bounded memory where it is easily wrong: batches of very many sequences, more work than a launch counts, accounts past four
gigabytes, threads with contexts of their own."""
import threading

import numpy as np
import pytest

from oracle import lm
from test_gpu_lm import Bed, from_bits, tables, to_bits
from test_gpu_lm_memory import (KINDS, Account, Moved, assert_codes, check_products, check_weights, free, normalisers, products, up, weights4,
                                weights_of)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpx):
    c = gpx.LmContext()
    yield c
    assert c.status() == (0, 0)
    c.free()


@pytest.mark.parametrize("seqs,most_new,most", [(2500, 1, 40), (4096, 1, 3), (700, 3, 50), (300, 33, 70)])
def test_batches_of_many_sequences(gpx, ctx, seqs, most_new, most):
    heads, kv, dim, page, dtype, keep = 2, 1, 64, 16, "bfloat16", 20
    rng = np.random.default_rng(seqs)
    context = rng.integers(1, most + 1, seqs)
    new = np.minimum(rng.integers(0, most_new + 1, seqs), context)
    new[0], context[0] = most_new, max(context[0], most_new)
    bed = Bed(gpx, new.tolist(), context.tolist(), heads, kv, dim, page, seed=1).upload()
    # ---- append at positions
    t = bed.tokens
    bits = to_bits(rng.standard_normal((t, (heads + 2 * kv) * dim)), dtype)
    vals = from_bits(bits, dtype)
    q, k, v = (vals[:, a * dim:b * dim].reshape(t, -1, dim) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    cos, sin = tables(30, dim)
    at, axis = rng.integers(0, 30, (t, 2)).astype(np.int32), np.arange(dim // 2) % 2
    lm.append(bed.k, bed.v, bed.ks, bed.vs, bed.table, bed.context, bed.first, lm.turn_at(k, at, axis, cos, sin, dim, False), v)
    turned = to_bits(lm.turn_at(q, at, axis, cos, sin, dim, False), dtype)
    dx, dcos, dsin, dat, dq = up(gpx, bits), up(gpx, cos), up(gpx, sin), up(gpx, at), gpx.DeviceBuffer(t * heads * dim * 2)
    base, width = dx.ptr.value, bits.shape[1]
    gpx.kv_append_at(bed.cache, bed.batch, base, base + 2 * heads * dim, base + 2 * (heads + kv) * dim, dq, heads, dtype, ctx,
                     gpx.Rope(dcos, dsin, 30, dim), gpx.KvPositions(dat, 2, axis), None, None, width, width, width)
    gpx.device_sync()
    assert np.array_equal(dq.download(np.uint16), turned.ravel())
    got = bed.download()
    for a, b in zip(got[:2], (bed.k, bed.v)):
        assert np.array_equal(np.where(a == 0x80, 0, a), np.where(b == 0x80, 0, b))
    assert np.array_equal(got[2], bed.ks) and np.array_equal(got[3], bed.vs)
    bed.k, bed.v = got[:2]
    # ---- accounts, choice, move
    q = from_bits(turned, dtype).reshape(t, heads, dim)
    lse = normalisers(q, bed, bed.context, True, 0)
    account, to_account, dl = Account(gpx, bed), Account(gpx, bed, seed=4), up(gpx, lse)
    want, bound = lm.weigh(account.w, account.slots, q, lse, bed.k, bed.ks, bed.table, bed.context, bed.first, decay=0.5)
    gpx.kv_weigh(bed.cache, bed.batch, dq, dl, account.handle, heads, dtype, ctx, decay=0.5)
    gpx.device_sync()
    weights = account.read()
    check_weights(weights, want, bound, account.w)
    kept, counts = up(gpx, np.zeros((seqs, kv, keep), np.int32)), up(gpx, np.zeros(seqs, np.int32))
    gpx.kv_choose(bed.batch, account.handle, kept, counts, keep, ctx, 2, 3)
    lists = lm.choose(weights, account.slots, bed.context, keep, 2, 3)
    to = Moved(gpx, bed, [x.shape[1] for x in lists], 32)
    gpx.kv_move(bed.cache, bed.batch, to.cache, to.dt, to.table.shape[1], kept, counts, keep, ctx, account.handle, to_account.handle)
    gpx.device_sync()
    have = kept.download(np.int32).reshape(seqs, kv, keep)
    for s, some in enumerate(lists):
        assert np.array_equal(have[s, :, :some.shape[1]], some)
    pages = [a.copy() for a in (to.k, to.v, to.ks, to.vs)]
    lm.move(bed.k, bed.v, bed.ks, bed.vs, bed.table, lists, *pages, to.table)
    assert_codes(to.download(), pages)
    assert ctx.status() == (0, 0)
    free(dx, dcos, dsin, dat, dq, dl, account, to_account, kept, counts, to, bed)


@pytest.mark.parametrize("new", [1, 90])
def test_more_work_than_a_launch_counts_is_reported(gpx, new):
    """Sequences as long as an int allows: nothing is read but their lengths."""
    mine = gpx.LmContext()
    kv, dim, page, heads, seqs = 128, 64, 16, 128, 2
    small = gpx.DeviceBuffer(1 << 20)
    cache = gpx.KvCache(4, page, kv, dim, small, small, small, small)
    longest = 2 ** 31 - 4097
    arrays = [up(gpx, a) for a in (np.zeros(4, np.int32), np.full(seqs, longest, np.int32), np.arange(seqs + 1, dtype=np.int32) * new)]
    batch = gpx.KvBatch(seqs, seqs * new, new, *arrays, 2 ** 27 + 8)
    account = gpx.KvWeights(small, seqs, kv, 2 ** 31)
    gpx.kv_weigh(cache, batch, small, small, account, heads, "bfloat16", mine)
    gpx.device_sync()
    assert mine.status() == (5, 0)
    mine.reset()
    counts = up(gpx, np.full(seqs, longest, np.int32))
    gpx.kv_move(cache, batch, cache, arrays[0], 2 ** 27 + 8, small, counts, 2 ** 31, mine)
    gpx.device_sync()
    assert mine.status() == (5, 0)
    mine.reset()
    one_more = up(gpx, np.full(seqs, longest + 1, np.int32))
    batch = gpx.KvBatch(seqs, seqs * new, new, arrays[0], one_more, arrays[2], 2 ** 27 + 8)
    gpx.kv_weigh(cache, batch, small, small, account, heads, "bfloat16", mine)
    gpx.device_sync()
    assert mine.status()[0] == 1
    cache.free(), mine.free()
    free(small, counts, one_more, *arrays)


def test_accounts_past_four_gigabytes(gpx, ctx):
    """Rows whose entries lie past 32 bits are added to, chosen from and moved; nothing else is initialised."""
    heads, kv, dim, page, dtype, context, keep, ld = 4, 1, 64, 16, "float16", [300, 80], 50, 700_000_000
    bed = Bed(gpx, [2, 1], context, heads, kv, dim, page, seed=3).upload()
    far = gpx.DeviceBuffer(2 * ld * 4)
    near = Account(gpx, bed)
    slots = up(gpx, np.array([1, 0], np.int32))
    account = gpx.KvWeights(far, 2, kv, ld, slots)
    for s, row in ((0, 1), (1, 0)):
        far.upload(near.w[near.slots[s], 0, :context[s]], offset=row * ld * 4)
    q = from_bits(to_bits(bed.rng.standard_normal((3, heads, dim)), dtype), dtype)
    dq, dl = up(gpx, to_bits(q, dtype)), up(gpx, normalisers(q, bed, context, True, 0))
    outs = []
    for a in (near.handle, account):
        kept, counts, to, after = gpx.DeviceBuffer(2 * keep * 4), gpx.DeviceBuffer(8), Moved(gpx, bed, [keep] * 2, page), Account(gpx, bed, seed=6)
        gpx.kv_weigh(bed.cache, bed.batch, dq, dl, a, heads, dtype, ctx)
        gpx.kv_choose(bed.batch, a, kept, counts, keep, ctx, 1, 5)
        gpx.kv_move(bed.cache, bed.batch, to.cache, to.dt, to.table.shape[1], kept, counts, keep, ctx, a, after.handle)
        gpx.device_sync()
        outs.append([kept.download(np.int32), counts.download(np.int32), *to.download(), after.read()])
        free(kept, counts, to, after)
    for a, b in zip(*outs):
        assert np.array_equal(a, b)
    for s, row in ((0, 1), (1, 0)):
        assert np.array_equal(far.download(np.float32, context[s], offset=row * ld * 4), near.read()[near.slots[s], 0, :context[s]])
    free(far, near, slots, dq, dl, bed)


def test_threads_with_contexts_of_their_own(gpx):
    """Products and accounts of several sizes at once, each thread on its stream with its context."""
    errors = []

    def work(seed):
        try:
            mine, stream, rng = gpx.LmContext(), gpx.Stream(0), np.random.default_rng(seed)
            for n, k, rows in ((9001 + seed, 4096, 1 + seed), (70, 256, 9), (6000, 5120, 20)):
                codes, scale_bits, z, w = weights4(rng, n, k, 64, True, "bfloat16")
                x = from_bits(to_bits(rng.standard_normal((rows, k)), "bfloat16"), "bfloat16")
                check_products(products(gpx, mine, x, codes, scale_bits, z, n, k, 64, "bfloat16", stream=stream), x, w, "bfloat16")
            for new in (1, 40):
                bed = Bed(gpx, [new] * (1 + 40 * seed % 100), [300] * (1 + 40 * seed % 100), 4, 2, 64, 16, seed=seed).upload()
                q = from_bits(to_bits(rng.standard_normal((bed.tokens, 4, 64)), "float16"), "float16")
                some = slice(0, 1)
                lse = np.zeros((bed.tokens, 4), np.float32) + 6
                account, dq, dl = Account(gpx, bed), up(gpx, to_bits(q, "float16")), up(gpx, lse)
                want, bound = lm.weigh(account.w, account.slots[some], q, lse, bed.k, bed.ks, bed.table[some], [300], bed.first[:2])
                gpx.kv_weigh(bed.cache, bed.batch, dq, dl, account.handle, 4, "float16", mine, stream=stream)
                stream.sync()
                row = account.slots[0]
                check_weights(account.read()[row:row + 1], want[row:row + 1], bound[row:row + 1], account.w[row:row + 1])
                free(account, dq, dl, bed)
            assert mine.status() == (0, 0)
            mine.free(), stream.destroy()
        except BaseException as e:  # noqa: BLE001 (a thread's failure is the test's)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


@pytest.mark.parametrize("new,heads", [(1, 4), (9, 4), (40, 2), (90, 4)])
@pytest.mark.parametrize("decay", [1.0, 0.5])
def test_pages_below_a_window_are_not_looked_up(gpx, ctx, new, heads, decay):
    """What no row sees may be another sequence's by now, or of no page: its accounts fade, and nothing is reported."""
    kv, dim, page, dtype, context, window = 1, 64, 16, "bfloat16", [500, 333], 70
    bed = Bed(gpx, [new, new], context, heads, kv, dim, page, seed=5).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    lse = normalisers(q, bed, context, True, window)
    for observed in (0, (new + 1) // 2):
        votes = observed or new
        table = bed.table.copy()
        for s, c in enumerate(context):
            below = max(0, c - votes + 1 - window) // page  # pages that end there
            table[s, :below] = [-1, bed.pages, 2 ** 31 - 1, -2 ** 31][s]
        bed.arrays[0].upload(table)
        account, dq, dl = Account(gpx, bed), up(gpx, to_bits(q, dtype)), up(gpx, lse)
        want, bound = lm.weigh(account.w, account.slots, q, lse, bed.k, bed.ks, bed.table, context, bed.first, None, True, window, observed, decay)
        gpx.kv_weigh(bed.cache, bed.batch, dq, dl, account.handle, heads, dtype, ctx, window=window, observed=observed, decay=decay)
        gpx.device_sync()
        check_weights(account.read(), want, bound, account.w)
        assert ctx.status() == (0, 0)
        free(account, dq, dl)
    bed.free()


@pytest.mark.parametrize("decay", [1.0, 0.5])
@pytest.mark.parametrize("case", [
    # new, context, page, window, observed; heads share keys four by four
    (1, 300, 16, 0, 0), (8, 300, 16, 0, 0),  # one pass over the rows
    (13, 300, 16, 0, 0), (16, 40, 16, 0, 0),  # two: a new token's key may be seen by rows of the second alone
    (13, 300, 64, 70, 0), (16, 500, 128, 100, 9), (16, 300, 32, 5, 12),  # a window's border in the middle of a page
    (20, 300, 16, 0, 0), (40, 300, 128, 33, 0), (90, 333, 64, 0, 30),  # many rows
], ids=lambda c: "%d-%d-p%d-w%d-o%d" % c)
def test_keys_of_pages_outside_the_cache_keep_their_accounts(gpx, case, decay):
    """Those that some row sees, however many rows there are and whichever of them see the key; the others fade as any do."""
    new, c, page, window, observed = case
    heads, kv, dim, dtype, context = 8, 2, 64, "bfloat16", [c, c - 7]
    mine = gpx.LmContext()
    bed = Bed(gpx, [new, new], context, heads, kv, dim, page, seed=6).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    dq, dl = up(gpx, to_bits(q, dtype)), up(gpx, normalisers(q, bed, context, True, window))
    lse = dl.download(np.float32).reshape(-1, heads)
    account = Account(gpx, bed)
    want, bound = lm.weigh(account.w, account.slots, q, lse, bed.k, bed.ks, bed.table, context, bed.first, None, True, window, observed, decay)
    votes = observed or new
    for s, n in enumerate(context):
        seen = max(0, n - votes + 1 - window) if window else 0
        last = (n - 1) // page
        for bad in sorted({seen // page, (n - new) // page, last // 2, last - 1, last} - {-1}):
            table = bed.table.copy()
            table[s, bad] = (-1, bed.pages, 2 ** 31 - 1, -2 ** 31)[(bad + s) % 4]
            bed.arrays[0].upload(table)
            account.dw.upload(account.w)
            gpx.kv_weigh(bed.cache, bed.batch, dq, dl, account.handle, heads, dtype, mine, window=window, observed=observed, decay=decay)
            gpx.device_sync()
            keys = slice(max(seen, bad * page), min(n, (bad + 1) * page))
            row = account.slots[s]
            expected, size = want.copy(), bound.copy()
            expected[row, :, keys], size[row, :, keys] = account.w[row, :, keys], 0
            got = account.read()
            assert np.array_equal(got[row, :, keys], account.w[row, :, keys]), (s, bad)
            check_weights(got, expected, size, account.w)
            assert mine.status() == ((2, s) if keys.start < keys.stop else (0, 0))
            mine.reset()
    mine.free()
    free(dq, dl, account, bed)


@pytest.mark.parametrize("keep,first,last", [(3000, 2, 100), (18000, 5, 0), (16390, 0, 7000)])
@pytest.mark.parametrize("kind", KINDS)
def test_batches_of_accounts_that_shared_memory_does_not_hold(gpx, ctx, kind, keep, first, last):
    """More accounts than a B200 has SMs, of more entries than 512 threads keep at once: they are read in pieces, and equal weights are
    counted across the ends of the pieces."""
    kv = 8
    context = [33000, 16384 + first + last, 16385 + first + last, 32768 + first + last, 32769 + first + last, 16383, 20000, 24001, 17, 3001,
               0, 31999, 18000, 18001, 16391, 25000, 30011, 19999, 28672, 1]
    context = [min(c, 33000) for c in context]
    rng = np.random.default_rng(keep)
    rows, ld = len(context) + 1, 33001
    w = weights_of(kind, (rows, kv, ld), rng)
    slots = rng.permutation(rows)[:len(context)].astype(np.int32)
    arrays = [up(gpx, a) for a in (np.full((len(context), 1), -9, np.int32), np.array(context, np.int32), np.full(len(context) + 1, -5, np.int32))]
    batch = gpx.KvBatch(len(context), 0, 0, *arrays, 1)
    dw, ds = up(gpx, w), up(gpx, slots)
    account = gpx.KvWeights(dw, rows, kv, ld, ds)
    kept, counts = up(gpx, np.full((len(context), kv, keep), -3, np.int32)), up(gpx, np.full(len(context), -3, np.int32))
    gpx.kv_choose(batch, account, kept, counts, keep, ctx, first=first, last=last)
    gpx.device_sync()
    got = kept.download(np.int32).reshape(len(context), kv, keep)
    assert counts.download(np.int32).tolist() == [min(c, keep) for c in context]
    for s, want in enumerate(lm.choose(w, slots, context, keep, first, last)):
        n = want.shape[1]
        assert np.array_equal(got[s, :, :n], want) and np.all(got[s, :, n:] == -3), s
    assert ctx.status() == (0, 0)
    free(dw, ds, kept, counts, *arrays)


def test_products_with_weights_that_are_gone_are_refused(gpx, ctx):
    codes, scales, zeros = (up(gpx, a) for a in (np.zeros((16, 32), np.uint8), np.zeros((16, 1), np.uint16), np.zeros((16, 1), np.uint8)))
    w, x, y = gpx.FourBit(codes, scales, zeros, 16, 64, 64, "bfloat16"), gpx.DeviceBuffer(128), gpx.DeviceBuffer(32)
    gpx.w4_matvec(w, x, y, 1, ctx)
    gpx.device_sync()
    w.free()
    with pytest.raises(Exception, match="packed"):
        gpx.w4_matvec(w, x, y, 1, ctx)
    w.free()
    free(codes, scales, zeros, x, y)
