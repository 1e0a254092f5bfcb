"""The decoder's serving step where it is easily wrong: threads with batches of their own, scales and scores far apart, pages below a
window, numbers at the ends of their types, more work than a launch counts."""
import threading

import numpy as np
import pytest

from oracle import lm
from test_gpu_lm import BITS, Bed, from_bits, preempted_runs, run_attention, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpx):
    c = gpx.LmContext()
    yield c
    assert c.status() == (0, 0)
    c.free()


def check(got, ref, weight, dtype, p_bits, score_err, keys, vmax):
    """What the formats allow: the result is rounded once; a factor of a product is rounded to `p_bits` bits and loses at most
    2^-31 of the largest; a score is off by `score_err`.  No absolute term: a result may be small as a whole."""
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    allowed = 1.01 * 2.0 ** -BITS[dtype] * np.abs(ref) + (2.0 ** -p_bits + 2 * score_err) * weight + 2.0 ** -31 * keys * vmax
    worst = np.max(np.abs(got.astype(np.float64) - ref) / allowed)
    assert worst <= 1, worst


def values_largest(bed):
    return float(np.max(np.abs(lm.decode(bed.v)).max((2, 3)) * bed.vs))


# ---- threads ----------------------------------------------------------------------------------------

def test_threads_with_batches_of_their_own(gpx):
    """Two tenants in two threads, whose launches of the same kernels need different amounts of shared memory."""
    heads, kv, dim, page, dtype = 8, 2, 128, 64, "bfloat16"
    turn, wrong = [threading.Semaphore(1), threading.Semaphore(0)], []

    def tenant(me, seqs):
        try:
            gpx.init_cuda(0)
            mine, s = gpx.LmContext(), gpx.Stream(0)
            bed = Bed(gpx, [2] * seqs, [40 + 3 * i for i in range(seqs)], heads, kv, dim, page, seed=seqs).upload()
            x = gpx.DeviceBuffer.from_numpy(to_bits(bed.rng.standard_normal((bed.tokens, (heads + 2 * kv) * dim)), dtype))
            q, out = (gpx.DeviceBuffer(bed.tokens * heads * dim * 2) for _ in range(2))
            at, ld, want = x.ptr.value, (heads + 2 * kv) * dim, None

            def step():
                gpx.kv_append(bed.cache, bed.batch, at, at + 2 * heads * dim, at + 2 * (heads + kv) * dim, q, heads, dtype, mine, None, None, s, ld, ld, ld)
                gpx.kv_attend(bed.cache, bed.batch, q, out, heads, dtype, mine, stream=s)
                s.sync()
                return out.download(np.uint16, stream=s)

            for i in range(600):
                if i < 6:  # (in turn, then as it comes)
                    turn[me].acquire()
                try:
                    got = step()
                finally:
                    if i < 6:
                        turn[1 - me].release()
                if i == 1:
                    want = got  # (the second append finds the scales of the first)
                if i > 1 and not np.array_equal(got, want):
                    wrong.append(f"step {i} of {seqs} sequences")
                    break
            if mine.status() != (0, 0):
                wrong.append(f"status {mine.status()}")
            for b in (x, q, out, mine, bed):
                b.free()
            s.destroy()
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
            turn[1 - me].release(6)

    threads = [threading.Thread(target=tenant, args=a) for a in ((0, 64), (1, 8))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


# ---- scales and scores far apart ---------------------------------------------------------------------

@pytest.mark.parametrize("new", [1, 3, 8, 20])
@pytest.mark.parametrize("power", [-8, 1, 3, 60])
def test_first_pages_of_zeros(gpx, ctx, new, power):
    """A page of zeros, as append stores it, before pages of any scale, with many blocks a tile."""
    seqs, c, heads, kv, dim, page, dtype = 48, 1200, 32, 8, 64, 16, "bfloat16"
    bed = Bed(gpx, [new] * seqs, [c] * seqs, heads, kv, dim, page, seed=new)
    bed.vs[:] = 2.0 ** power
    bed.v[bed.table[:, 0]], bed.vs[bed.table[:, 0]] = 0, 2.0 ** -126
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads)
    some = 4 * new
    ref, ref_lse, weight = lm.attend(q[:some], bed.k, bed.v, bed.ks, bed.vs, bed.table, bed.context[:4], bed.first[:5])
    check(got[:some], ref, weight, dtype, 11, 2.0 ** -14, c, values_largest(bed))
    assert np.all(np.abs(lse[:some] - ref_lse) <= 2.0 ** -14)
    bed.free()


@pytest.mark.parametrize("new", [4, 8])
@pytest.mark.parametrize("power", [-8, 3, 100])
def test_rows_that_do_not_see_a_page_of_zeros(gpx, ctx, new, power):
    """A page of zeros at the lower end of a window: the later of the new tokens see none of it, and have no sum when the scale grows."""
    seqs, c, heads, kv, dim, page, dtype, window = 40, 1000, 32, 8, 64, 16, "bfloat16", 900
    bed = Bed(gpx, [new] * seqs, [c + i for i in range(seqs)], heads, kv, dim, page, seed=new)
    bed.vs[:] = 2.0 ** power
    for s in range(seqs):
        first = bed.table[s, (c + s - new + 1 - window) // page]
        bed.v[first], bed.vs[first] = 0, 2.0 ** -126
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, window=window)
    some = 16 * new
    ref, ref_lse, weight = lm.attend(q[:some], bed.k, bed.v, bed.ks, bed.vs, bed.table, bed.context[:16], bed.first[:17], window=window)
    check(got[:some], ref, weight, dtype, 11, 2.0 ** -14, c, values_largest(bed))
    assert np.all(np.abs(lse[:some] - ref_lse) <= 2.0 ** -14)
    bed.free()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_page_of_zeros_does_not_hide_what_other_warps_see(gpx, ctx, dim):
    """One key 2^10 ahead of 1 200 others that weigh as much together, in the sixteen keys of a block whose first page is zeros."""
    seqs, c, heads, kv, page, dtype = 48, 1200, 16, 8, 16, "bfloat16"
    bed = Bed(gpx, [1] * seqs, [c] * seqs, heads, kv, dim, page, seed=dim)
    bed.vs[:] = 2.0 ** -8
    bed.v[bed.table[:, 0]], bed.vs[bed.table[:, 0]] = 0, 2.0 ** -126
    bed.k[..., 0], bed.ks[:] = 0, 1.0
    bed.k[bed.table[:, 12], :, 2, 0] = 0x7E  # 448, key 194 of each
    bed.upload()
    q = np.zeros((bed.tokens, heads, dim), np.float32)
    q[..., 0] = 1
    scale = float(np.float32(10 * np.log(2) / 448))
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, scale=scale)
    ref, ref_lse, weight = lm.attend(q[:4], bed.k, bed.v, bed.ks, bed.vs, bed.table, bed.context[:4], bed.first[:5], scale)
    check(got[:4], ref, weight, dtype, 11, 2.0 ** -17, c, values_largest(bed))
    assert np.all(np.abs(lse[:4] - ref_lse) <= 2.0 ** -17)
    bed.free()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new,seqs", [(1, 444), (5, 444), (40, 148)])
def test_a_first_key_that_holds_most_of_the_weight(gpx, ctx, dtype, new, seqs):
    """Sixty thousand keys of 2^-25.6 each behind it, with values 448 times its own: they are a third of the result."""
    c, heads, kv, dim, page = 60000, 1, 1, 64, 128
    bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=1)
    bed.k[:], bed.v[:], bed.ks[:], bed.vs[:] = 0, 0x7E, 1.0, 1.0
    bed.k[bed.table[0, 0], 0, 0, 0], bed.v[bed.table[0, 0], 0, 0] = 0x7E, 0x38  # 448, and 1
    # (all sequences have the same pages)
    bed.table = np.repeat(bed.table, seqs, 0)
    bed.new, bed.context, bed.tokens = [new] * seqs, np.full(seqs, c, np.int32), new * seqs
    bed.first = (np.arange(seqs + 1) * new).astype(np.int32)
    bed.upload()
    q = np.zeros((bed.tokens, heads, dim), np.float32)
    q[..., 0] = 1
    scale = float(np.float32(25.6 * np.log(2) / 448))
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, causal=False, scale=scale)
    ref, ref_lse, weight = lm.attend(q[:1], bed.k, bed.v, bed.ks, bed.vs, bed.table[:1], [c], [0, 1], scale, causal=False)
    check(got, np.broadcast_to(ref, got.shape), np.broadcast_to(weight, got.shape), dtype, 11, 2.0 ** -17, c, 448.0)
    assert np.all(np.abs(lse - ref_lse[0, 0]) <= 2.0 ** -17)
    bed.free()


# ---- pages that nothing can see -----------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["returned", "of others", "small values"])
@pytest.mark.parametrize("new,context,window,page", [([1, 1], [777, 300], 50, 16), ([4, 1], [900, 64], 37, 32), ([30, 8], [700, 129], 20, 16),
                                                     ([80, 100], [815, 333], 100, 32), ([300, 40], [1300, 1000], 33, 16), ([1] * 100, [1000 + i for i in range(100)], 300, 16)])
def test_pages_below_a_window_have_no_influence(gpx, ctx, kind, new, context, window, page):
    """Pages that no row sees any more: taken out of the table, or somebody else's by now; and the other values as small as they go."""
    heads, kv, dim, dtype = 4, 2, 128, "bfloat16"
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=window)
    if kind == "small values":
        bed.vs = np.ldexp(bed.vs, -80)
    want = [a.copy() for a in (bed.k, bed.v, bed.ks, bed.vs, bed.table)]
    for s, (n, c) in enumerate(zip(new, context)):
        dead = max(0, c - n + 1 - window) // page
        if kind == "returned":
            bed.table[s, :dead] = -1
        else:
            bed.v[bed.table[s, :dead]], bed.k[bed.table[s, :dead]] = 0x7F, 0x7F
            bed.vs[bed.table[s, :dead]], bed.ks[bed.table[s, :dead]] = 2.0 ** 100, 2.0 ** 90
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, window=window)
    status = ctx.status()
    ctx.reset()
    assert status == (0, 0)
    ref, ref_lse, weight = lm.attend(q, *want, bed.context, bed.first, None, True, window)
    bed.v, bed.vs = want[1], want[3]
    check(got, ref, weight, dtype, 11, 2.0 ** -13, max(context), values_largest(bed))
    assert np.all(np.abs(lse - ref_lse) <= 2.0 ** -13)
    bed.free()


@pytest.mark.parametrize("new,context", [(200, 150), (20, 13), (200, 190), (300, 40)])
def test_the_largest_window_is_no_window(gpx, ctx, new, context):
    """More new tokens than keys: the first rows' positions are negative."""
    heads, kv, dim, page, dtype = 4, 2, 64, 16, "bfloat16"
    bed = Bed(gpx, [new], [context], heads, kv, dim, page, seed=new).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((new, heads, dim)), dtype), dtype)
    want = run_attention(gpx, ctx, bed, q, dtype, heads)
    got = run_attention(gpx, ctx, bed, q, dtype, heads, window=2 ** 31 - 1)
    ref, _, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, [context], bed.first)
    for out, lse in (want, got):
        assert np.array_equal(np.isneginf(lse), np.isneginf(want[1]))
        seen = np.abs(ref).sum(-1) > 0
        assert np.all(out[~seen] == 0)
        check(out[seen], ref[seen], weight[seen], dtype, 11, 2.0 ** -13, context, values_largest(bed))
    bed.free()


# ---- the ends of the types ----------------------------------------------------------------------------

@pytest.mark.parametrize("new", [1, 8, 40])
@pytest.mark.parametrize("power", [-120, -24, -21])
def test_tiny_queries_over_keys_of_zero(gpx, ctx, new, power):
    """Scores are zero: a row's result is the mean of what it sees, hidden keys or not."""
    c, heads, kv, dim, page, dtype = 100 + new, 4, 2, 64, 64, "bfloat16"
    bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=new)
    bed.k[:], bed.ks[:] = 0, 2.0 ** -126
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((new, heads, dim)) * 2.0 ** power, dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads)
    ref, ref_lse, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, [c], bed.first)
    check(got, ref, weight, dtype, 11, 2.0 ** -19, c, values_largest(bed))
    assert np.all(np.abs(lse - ref_lse) <= 2.0 ** -19)
    bed.free()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("power", [-127, 125, 126, 127])
def test_queries_at_the_ends_of_their_type(gpx, ctx, new, power):
    """Rows whose largest element is of either end, with keys' scales that bring the scores back to a few units."""
    c, heads, kv, dim, page, dtype = 100 + new, 4, 2, 128, 64, "bfloat16"
    bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=new)
    bed.ks[:] = 2.0 ** (-10 - power if power > 0 else 118)
    bed.upload()
    x = np.clip(bed.rng.standard_normal((new, heads, dim)), -1.9, 1.9).astype(np.float64)
    q = from_bits(to_bits((x * 2.0 ** power).astype(np.float32), dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads)
    ref, ref_lse, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, [c], bed.first)
    check(got, ref, weight, dtype, 11, 2.0 ** -13, c, values_largest(bed))
    assert np.all(np.abs(lse - ref_lse) <= 2.0 ** -13)
    bed.free()


# ---- more work than a launch counts -------------------------------------------------------------------

@pytest.mark.parametrize("seqs,new,pages_a_seq", [(8, 1, 1 << 13), (4, 1, 1 << 13), (32, 1, 1 << 12), (1, 1, 1 << 15), (1, 33, 1 << 16), (2, 33, 1 << 16)])
def test_more_work_than_a_launch_counts_is_reported(gpx, seqs, new, pages_a_seq):
    """Sums over the sequences that pass 31 bits, of one warp's sequences or of one sequence alone: nothing is done.
    (All sequences have the one page of the cache, again and again.)"""
    heads, dim, page = 1 << 15, 64, 128
    mine, cache = gpx.LmContext(), gpx.KvCache(1, page, heads, dim)
    d = gpx.DeviceBuffer.from_numpy
    arrays = [d(np.zeros((seqs, pages_a_seq), np.int32)), d(np.full(seqs, pages_a_seq * page, np.int32)), d((np.arange(seqs + 1) * new).astype(np.int32))]
    batch = gpx.KvBatch(seqs, seqs * new, new, *arrays, pages_a_seq)
    q, out = gpx.DeviceBuffer(seqs * new * heads * dim * 2), d(np.full(seqs * new * heads * dim, 0x1234, np.uint16))
    q.zero()
    gpx.kv_attend(cache, batch, q, out, heads, "bfloat16", mine)
    gpx.device_sync()
    assert mine.status() == (5, 0)
    assert np.all(out.download(np.uint16) == 0x1234)
    for b in (*arrays, q, out, mine, cache):
        b.free()


@pytest.mark.parametrize("new", [1, 40])
def test_sequences_at_the_end_of_an_int_are_reported(gpx, new):
    """The places of the last page's end and of what is fetched ahead have to be ints; what does not fit counts as empty."""
    heads, dim, page, pages_a_seq = 1, 64, 128, 1 << 24
    mine, cache = gpx.LmContext(), gpx.KvCache(1, page, heads, dim)
    d = gpx.DeviceBuffer.from_numpy
    for context in (2 ** 31 - 4096, 2 ** 31 - 64, 2 ** 31 - 1):
        arrays = [d(np.zeros((1, pages_a_seq), np.int32)), d(np.array([context], np.int32)), d(np.array([0, new], np.int32))]
        batch = gpx.KvBatch(1, new, new, *arrays, pages_a_seq)
        x, out = gpx.DeviceBuffer(new * heads * dim * 2), d(np.full(new * heads * dim, 0x1234, np.uint16))
        x.zero()
        gpx.kv_attend(cache, batch, x, out, heads, "bfloat16", mine)
        gpx.device_sync()
        assert mine.status() == (1, 0)
        mine.reset()
        gpx.kv_append(cache, batch, None, x, x, None, heads, "bfloat16", mine)
        gpx.device_sync()
        assert mine.status() == (1, 0)
        mine.reset()
        assert np.all(out.download(np.uint16) == 0x1234) and not cache.k_scale.download(np.float32).any()
        for b in (*arrays, x, out):
            b.free()
    mine.free(), cache.free()


# ---- paths that ordinary sizes do not take --------------------------------------------------------------

@pytest.mark.parametrize("seqs", [127, 128, 300])
@pytest.mark.parametrize("most", [20, 300])
def test_prompts_of_many_sequences(gpx, ctx, seqs, most):
    """Sums over more than 127 sequences lie in the context; units of a few blocks are tiles, longer ones are cut."""
    heads, kv, dim, page, dtype = 8, 2, 64, 32, "bfloat16"
    new = [(7 * i) % most if i % 5 else 0 for i in range(seqs - 1)] + [most]
    context = [n + (i * 131) % 2500 for i, n in enumerate(new)]
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=seqs).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads)
    for some in (slice(0, 4), slice(seqs - 3, seqs)):
        rows = slice(bed.first[some.start], bed.first[some.stop])
        ref, ref_lse, weight = lm.attend(q[rows], bed.k, bed.v, bed.ks, bed.vs, bed.table[some], bed.context[some], bed.first[some.start:some.stop + 1] - rows.start)
        check(got[rows], ref, weight, dtype, 11, 2.0 ** -13, max(context), values_largest(bed))
        assert np.all(np.abs(lse[rows] - ref_lse) <= 2.0 ** -13)
    # (the other kernel, a sequence at a time, on all of the rest)
    again = np.zeros_like(got)
    for s in range(seqs):
        if new[s] == 0:
            continue
        arrays = [gpx.DeviceBuffer.from_numpy(a) for a in (bed.table[s:s + 1], bed.context[s:s + 1], np.array([0, new[s]], np.int32))]
        rows = slice(bed.first[s], bed.first[s + 1])
        alone = type("Alone", (), {"cache": bed.cache, "tokens": new[s], "dim": dim, "batch": gpx.KvBatch(1, new[s], new[s], *arrays, bed.table.shape[1])})
        again[rows], _ = run_attention(gpx, ctx, alone, q[rows], dtype, heads)
        for a in arrays:
            a.free()
    # two results within a rounding each, and their factors'
    assert np.all(np.abs(got - again) <= 2.0 ** -7 * np.abs(again) + 2.0 ** -9 * values_largest(bed))
    bed.free()


@pytest.mark.parametrize("new,context,heads,kv,dim,dtype,causal,window,run_us", [
    ([5] * 60, [4000 + 31 * i for i in range(60)], 16, 4, 128, "float16", True, 0, 250),      # two tiles of rows
    ([8] * 60, [4000 + 31 * i for i in range(60)], 16, 4, 64, "bfloat16", True, 3000, 250),   # four
    ([1] * 64, [6000] * 64, 16, 4, 128, "float16", True, 2500, 100),
    ([64] * 90, [700] * 90, 16, 8, 64, "bfloat16", True, 0, 100),                            # units that are tiles as they are
    ([37] * 100, [512] * 100, 12, 12, 64, "float16", False, 0, 100),
    ([900, 500], [4000, 2500], 16, 4, 128, "float16", True, 0, 200),
    ([700, 900], [3000, 900], 16, 4, 64, "bfloat16", True, 600, 100),
    ([300, 700], [3000, 2000], 16, 4, 128, "bfloat16", False, 0, 200),
    ([40] * 200, [60 + 17 * i for i in range(200)], 8, 2, 64, "bfloat16", True, 0, 100),      # sums in the context
])
def test_attention_of_every_kind_drains_and_resumes_bit_identically(gpx, ctx, new, context, heads, kv, dim, dtype, causal, window, run_us):
    page = 64
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=4).upload()
    q = to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype)
    dq = gpx.DeviceBuffer.from_numpy(q)
    out, lse = gpx.DeviceBuffer(bed.tokens * heads * dim * 2), gpx.DeviceBuffer(bed.tokens * heads * 4)

    def fresh():
        out.zero(), lse.zero()

    want = preempted_runs(gpx, lambda blp, s: gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, dtype, ctx, causal=causal, window=window, lse=lse, blp=blp, stream=s),
                          lambda: [out.download(np.uint16), lse.download(np.uint32)], fresh, run_us, at_least=1)
    # a launch without a word gives the same numbers within a rounding of each
    got, _ = run_attention(gpx, ctx, bed, from_bits(q, dtype), dtype, heads, causal=causal, window=window)
    other = from_bits(want[0], dtype).reshape(got.shape)
    assert np.all(np.abs(got - other) <= 2.0 ** (1 - BITS[dtype]) * np.abs(got) + 2.0 ** -9 * values_largest(bed) * (8 if dtype == "bfloat16" else 1))
    dq.free(), out.free(), lse.free(), bed.free()


@pytest.mark.parametrize("new,p_bits", [(1, 20), (5, 20), (32, 20), (40, 11)])
def test_factors_of_float16_results(gpx, ctx, new, p_bits):
    """Values of both signs that nearly cancel show the factors' bits: 22 up to 32 rows a head of keys, 11 beyond."""
    heads, kv, dim, page, dtype = 1, 1, 64, 64, "float16"
    for c in (2, 3, 5, 33):
        bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=c)
        bed.v[:] = np.where(np.arange(page)[:, None] % 2, 0x7E, 0xFE)  # 448 and -448
        bed.vs[:], bed.ks[:] = 1.0, 2.0 ** -10
        bed.upload()
        q = from_bits(to_bits(bed.rng.standard_normal((new, heads, dim)), dtype), dtype)
        got, _ = run_attention(gpx, ctx, bed, q, dtype, heads, causal=False)
        ref, _, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, [c], bed.first, causal=False)
        # scores below 1: float sums of 64 products, the factor and the exponential are good to 2^-21
        check(got, ref, weight, dtype, p_bits, 2.0 ** -21, c, 448.0)
        bed.free()
