"""The decoder's serving step on the GPU against its restatement in 64 bits: cache append with rotation, attention over
the paged 8-bit cache, token scores; their refusals, what they report, and preemption."""
import ctypes
import time

import numpy as np
import pytest

from oracle import lm

pytestmark = pytest.mark.gpu


# ---- 16-bit formats ---------------------------------------------------------------------------------

def to_bits(x, dtype):
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "float32":
        return x
    if dtype == "float16":
        with np.errstate(all="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def from_bits(b, dtype):
    if dtype == "float32":
        return b
    if dtype == "float16":
        return b.view(np.float16).astype(np.float32)
    return (b.astype(np.uint32) << 16).view(np.float32)


BITS = {"bfloat16": 8, "float16": 11}  # significant bits of a result


class Bed:
    """A pool with shuffled pages, a ragged batch over it, and the same in numpy."""

    def __init__(self, gpx, new, context, heads, kv_heads, dim, page, seed=0, spare=3, garbage=None):
        rng = np.random.default_rng(seed)
        self.gpx, self.rng = gpx, rng
        self.new, self.heads, self.kv, self.dim, self.page = new, heads, kv_heads, dim, page
        self.context = np.array(context, np.int32)
        self.first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.first[-1])
        per = [-(-c // page) for c in context]
        pages = sum(per) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(context), max(1, max(per))), -7, np.int32)  # (entries past a sequence are not looked at)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.k, self.v = (self._codes(pages, garbage) for _ in range(2))
        self.ks, self.vs = (np.ldexp(1.0, rng.integers(-9, -4, (pages, kv_heads))).astype(np.float32) for _ in range(2))
        if garbage is not None:
            # slots past a sequence's end and pages of nobody hold anything, NaN codes too
            used = np.zeros((pages, page), bool)
            for s, c in enumerate(context):
                for j in range(c):
                    used[self.table[s, j // page], j % page] = True
            for x in (self.k, self.v):
                x[:] = np.where(used[:, None, :, None], x, garbage)
        self.pages = pages

    def _codes(self, pages, garbage):
        if pages * self.kv * self.page * self.dim > 1 << 24:  # (any finite codes: quickly made)
            x = self.rng.integers(0, 256, (pages, self.kv, self.page, self.dim), np.uint8)
            return np.where(x & 0x7F == 0x7F, np.uint8(0), x)
        x = self.rng.standard_normal((pages, self.kv, self.page, self.dim)) * 100
        return lm.encode(np.clip(x, -448, 448))

    def upload(self):
        D = self.gpx.DeviceBuffer.from_numpy
        self.dk, self.dv, self.dks, self.dvs = D(self.k), D(self.v), D(self.ks), D(self.vs)
        self.cache = self.gpx.KvCache(self.pages, self.page, self.kv, self.dim, self.dk, self.dv, self.dks, self.dvs)
        self.arrays = D(self.table), D(self.context), D(self.first)
        self.batch = self.gpx.KvBatch(len(self.new), self.tokens, int(max(self.new)), *self.arrays, self.table.shape[1])
        return self

    def download(self):
        shape = self.k.shape
        return (self.dk.download(np.uint8).reshape(shape), self.dv.download(np.uint8).reshape(shape),
                self.dks.download(np.float32).reshape(self.ks.shape), self.dvs.download(np.float32).reshape(self.ks.shape))

    def free(self):
        self.cache.free()
        for b in (self.dk, self.dv, self.dks, self.dvs, *self.arrays):
            b.free()


def tables(positions, rotated):
    half = max(1, rotated // 2)
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(half) / half)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@pytest.fixture(scope="module")
def ctx(gpx):
    c = gpx.LmContext()
    yield c
    assert c.status() == (0, 0)
    c.free()


# ---- append -----------------------------------------------------------------------------------------

APPENDS = [
    # new tokens, tokens in all, heads, kv_heads, dim, page, dtype, rotated, paired
    ([1], [1], 2, 2, 64, 16, "bfloat16", 64, False),
    ([1], [129], 32, 8, 128, 64, "bfloat16", 128, False),
    ([1, 0, 1, 1], [17, 5, 16, 1], 6, 2, 64, 16, "float16", 64, True),
    ([1] * 67, list(range(1, 68)), 5, 5, 128, 32, "bfloat16", 64, False),
    ([0, 3, 0], [0, 3, 9], 4, 1, 64, 32, "float16", 0, False),
    ([5, 1, 16, 17, 33], [5, 130, 16, 40, 33], 8, 4, 128, 16, "float16", 128, True),
    ([7, 300, 64], [20, 300, 128], 4, 2, 64, 64, "bfloat16", 32, True),
    ([2, 129, 256, 200], [130, 129, 256, 327], 8, 2, 128, 128, "bfloat16", 128, False),
    ([2, 140], [66, 400], 3, 3, 64, 128, "float16", 8, False),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "%dx%d-%d-%d-p%d-%s-r%d%s" % (len(c[0]), max(c[0]), c[3], c[4], c[5], c[6], c[7], "p" * c[8]))
@pytest.mark.parametrize("kind", ["plain", "strided", "wild"])
def test_append_is_the_definition_bit_for_bit(gpx, ctx, case, kind):
    new, context, heads, kv, dim, page, dtype, rotated, paired = case
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=len(new) + dim).upload()
    rng, t = bed.rng, bed.tokens
    # strided: one projection's output holds queries, keys and values side by side, and queries are turned in place
    width = (heads + 2 * kv) * dim + (12 if kind == "strided" else 0)
    x = rng.standard_normal((t, width)) * np.exp(rng.standard_normal((t, 1)) * (3.0 if kind == "wild" else 0.3))
    if kind == "wild":
        # zeros, numbers that are not finite, the largest and the smallest of the type
        x[rng.random(x.shape) < 0.02] = 0
        x[rng.random(x.shape) < 0.005] = np.nan
        x[rng.random(x.shape) < 0.005] = -np.inf
        x[rng.random((t, 1)).repeat(width, 1) < 0.1] = 0
        x[0, -dim:] = 6e4 if dtype == "float16" else 3e38
    bits = to_bits(x, dtype)
    vals = from_bits(bits, dtype)
    q = vals[:, :heads * dim].reshape(t, heads, dim)
    k = vals[:, heads * dim:(heads + kv) * dim].reshape(t, kv, dim)
    v = vals[:, (heads + kv) * dim:(heads + 2 * kv) * dim].reshape(t, kv, dim)
    cos, sin = tables(max(context) + 2, rotated)
    want = [a.copy() for a in (bed.k, bed.v, bed.ks, bed.vs)]
    lm.append(*want, bed.table, bed.context, bed.first, k, v, cos, sin, rotated, paired)
    pos = np.concatenate([np.arange(c - n, c) for n, c in zip(new, context)])
    want_q = to_bits(lm.turn(q, pos, cos, sin, rotated, paired), dtype).reshape(t, -1)

    d = gpx.DeviceBuffer.from_numpy
    dx, dcos, dsin = d(bits), d(cos), d(sin)
    rope = gpx.Rope(dcos, dsin, cos.shape[0], rotated, paired) if rotated else None
    s = gpx.Stream(0)
    base = dx.ptr.value
    args = [base, base + 2 * heads * dim, base + 2 * (heads + kv) * dim]
    if kind == "strided":
        gpx.kv_append(bed.cache, bed.batch, args[0], args[1], args[2], args[0], heads, dtype, ctx, rope, None, s, width, width, width, width)
        s.sync()
        got_q = dx.download(np.uint16).reshape(t, width)
        assert np.array_equal(got_q[:, heads * dim:], bits[:, heads * dim:])
        got_q = got_q[:, :heads * dim]
    else:
        out = gpx.DeviceBuffer(t * heads * dim * 2)
        gpx.kv_append(bed.cache, bed.batch, args[0], args[1], args[2], out, heads, dtype, ctx, rope, None, s, width, width, width)
        s.sync()
        got_q = out.download(np.uint16).reshape(t, heads * dim)
        out.free()
    nan_q = np.isnan(from_bits(want_q, dtype))
    assert np.array_equal(np.isnan(from_bits(got_q, dtype)), nan_q)
    assert np.array_equal(got_q[~nan_q], want_q[~nan_q])
    for name, got, ref in zip(("k", "v", "k_scale", "v_scale"), bed.download(), want):
        if got.dtype == np.uint8:
            got, ref = np.where(got & 0x7F == 0x7F, 0x7F, got), np.where(ref & 0x7F == 0x7F, 0x7F, ref)  # (a NaN has no sign)
            got, ref = np.where(got == 0x80, 0, got), np.where(ref == 0x80, 0, ref)
        assert np.array_equal(got, ref), name
    assert ctx.status() == (0, 0)
    for b in (dx, dcos, dsin):
        b.free()
    bed.free(), s.destroy()


def test_append_token_by_token_and_without_queries(gpx, ctx):
    """A page that gains larger and larger tokens rounds what it holds again; keys and values alone can be appended."""
    n, kv, dim, page = 40, 2, 64, 16
    bed = Bed(gpx, [1], [1], kv, kv, dim, page, spare=4)
    bed.table = np.array([[2, 0, 4, 1]], np.int32)
    bed.upload()
    want = [a.copy() for a in (bed.k, bed.v, bed.ks, bed.vs)]
    cos, sin = tables(n, dim)
    dcos, dsin = gpx.DeviceBuffer.from_numpy(cos), gpx.DeviceBuffer.from_numpy(sin)
    rope = gpx.Rope(dcos, dsin, n, dim)
    x = bed.rng.standard_normal((n, 2, kv, dim)) * np.exp2(np.arange(n) % page - 8)[:, None, None, None]
    for i in range(n):
        bits = to_bits(x[i].reshape(2, -1), "bfloat16")
        kv_now = from_bits(bits, "bfloat16").reshape(2, 1, kv, dim)
        dx = gpx.DeviceBuffer.from_numpy(bits)
        bed.arrays[1].upload(np.array([i + 1], np.int32))
        gpx.kv_append(bed.cache, bed.batch, None, dx, dx.ptr.value + 2 * kv * dim, None, kv, "bfloat16", ctx, rope)
        gpx.device_sync()
        lm.append(*want, bed.table, [i + 1], [0, 1], kv_now[0], kv_now[1], cos, sin, dim, False)
        dx.free()
    for got, ref in zip(bed.download(), want):
        assert np.array_equal(got, ref)
    bed.free(), dcos.free(), dsin.free()


# ---- attend -----------------------------------------------------------------------------------------

def check_attention(got, lse, ref, ref_lse, weight, dtype, keys, vmax, score_size):
    """Bounds of what the formats allow: the result is rounded once; probabilities have 12 bits of rounding where the
    result has eight (and an absolute one of half precision's smallest steps), 22 where it has eleven; scores and exponentials are float."""
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(got), nan)
    p_round = 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -20
    score_err = 2.0 ** -17 * (1 + score_size)
    allowed = 1.01 * 2.0 ** -BITS[dtype] * np.abs(ref) + (p_round + score_err) * weight + 2.0 ** -24 * keys * vmax + 2.0 ** -24
    err = np.abs(got.astype(np.float64) - ref)
    worst = np.nanmax(np.where(nan, 0, err / allowed), initial=0)
    assert worst <= 1, worst
    if lse is not None:
        assert np.array_equal(np.isneginf(lse), np.isneginf(ref_lse)) and np.array_equal(np.isnan(lse), np.isnan(ref_lse))
        fine = np.isfinite(ref_lse)
        assert np.all(np.abs(lse[fine] - ref_lse[fine]) <= score_err), np.max(np.abs(lse[fine] - ref_lse[fine]))


def run_attention(gpx, ctx, bed, q, dtype, heads, blp=None, stream=None, with_lse=True, **kw):
    d = gpx.DeviceBuffer.from_numpy
    dq = d(to_bits(q, dtype))
    out, lse = gpx.DeviceBuffer(max(16, bed.tokens * heads * bed.dim * 2)), gpx.DeviceBuffer(max(16, bed.tokens * heads * 4))
    gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, dtype, ctx, lse=lse if with_lse else None, blp=blp, stream=stream, **kw)
    gpx.device_sync()
    got = from_bits(out.download(np.uint16, bed.tokens * heads * bed.dim), dtype).reshape(bed.tokens, heads, bed.dim)
    got_lse = lse.download(np.float32, bed.tokens * heads).reshape(bed.tokens, heads)
    for b in (dq, out, lse):
        b.free()
    return got, got_lse


ATTENDS = [
    # new, context, heads, kv_heads, dim, page, dtype, causal, window
    ([1], [1], 1, 1, 64, 16, "bfloat16", True, 0),
    ([1], [64], 32, 8, 128, 64, "bfloat16", True, 0),
    ([1], [65], 8, 8, 128, 128, "float16", True, 0),
    ([1, 1, 0, 1, 1], [15, 16, 7, 17, 0], 4, 2, 64, 16, "float16", True, 0),
    ([1] * 9, [1, 31, 32, 33, 63, 127, 128, 129, 500], 16, 1, 128, 32, "bfloat16", True, 0),
    ([1], [4099], 16, 2, 64, 128, "bfloat16", True, 0),
    ([1, 1], [777, 300], 28, 4, 128, 16, "float16", True, 50),
    ([3, 1, 5], [3, 90, 200], 6, 6, 64, 32, "bfloat16", True, 0),
    ([5, 4], [2, 300], 12, 4, 64, 64, "float16", True, 0),  # more new tokens than keys: the first rows see none
    ([7, 2], [300, 70], 24, 2, 64, 16, "bfloat16", True, 33),
    ([37, 5], [37, 260], 8, 2, 128, 64, "float16", True, 0),
    ([70, 130, 1], [140, 130, 513], 4, 1, 128, 32, "bfloat16", True, 64),
    ([9, 40], [70, 1], 4, 2, 64, 128, "float16", False, 0),
    ([100], [1000], 5, 5, 128, 128, "bfloat16", True, 1),
    ([200, 3], [200, 900], 6, 3, 64, 16, "bfloat16", True, 0),
    ([129, 260], [515, 260], 8, 2, 128, 128, "bfloat16", False, 0),
    ([300, 17], [700, 640], 12, 12, 64, 64, "float16", True, 100),
]


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "%dx%d-%d-%d.%d-%d-p%d-%s-%d-w%d" % (len(c[0]), max(c[0]), max(c[1]), *c[2:]))
def test_attention_matches_the_definition(gpx, ctx, case):
    new, context, heads, kv, dim, page, dtype, causal, window = case
    # what lies past a sequence's end: NaN codes
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=7, garbage=0xFF).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)) * 2, dtype), dtype)
    got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, causal=causal, window=window)
    ref, ref_lse, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, context, bed.first, None, causal, window)
    check_attention(got, lse, ref, ref_lse, weight, dtype, max(context), 448 * 2.0 ** -5, 60)
    assert ctx.status() == (0, 0)
    # the same again without the normalisers: the same bits, nothing is left behind in the context
    again, _ = run_attention(gpx, ctx, bed, q, dtype, heads, causal=causal, window=window, with_lse=False)
    assert np.array_equal(again, got)
    bed.free()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim,new", [(128, 6), (64, 6), (128, 150), (64, 150)])
def test_what_is_not_finite_reaches_the_rows_that_see_it_only(gpx, ctx, dtype, dim, new):
    n, c, heads, kv, page = new, new + 64, 4, 2, 32
    bed = Bed(gpx, [n, 2], [c, 40], heads, kv, dim, page, seed=3)
    for j, where in ((c - 3, "v"), (c - n // 2, "v"), (c - 2, "k"), (c - n - 5, "v")):  # new tokens and an old one
        codes = bed.k if where == "k" else bed.v
        codes[bed.table[0, j // page], 1 if j == c - 3 else 0, j % page, 5 + j % 7] = 0x7F if j % 2 else 0xFF
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), dtype), dtype).copy()
    q[1, 3, 2], q[n, 0, 7] = np.inf, np.nan
    for window in (0, 4):
        got, lse = run_attention(gpx, ctx, bed, q, dtype, heads, window=window)
        ref, ref_lse, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, [c, 40], bed.first, None, True, window)
        assert np.isnan(ref).any() and not np.isnan(ref).all()
        check_attention(got, lse, ref, ref_lse, weight, dtype, c, 448 * 2.0 ** -5, 60)
    bed.free()


@pytest.mark.parametrize("new", [1, 40])
def test_scales_of_any_size(gpx, ctx, new):
    """Pages whose values' scales lie far apart, queries far from one, a scale of the caller's, padded rows."""
    c, heads, kv, dim, page, dtype = 1000 + new, 4, 2, 128, 16, "bfloat16"
    bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=5)
    bed.vs = np.ldexp(1.0, bed.rng.integers(-30, 20, bed.vs.shape)).astype(np.float32)
    bed.vs[bed.table[0, 3]] = 2.0 ** -126
    bed.ks = np.full_like(bed.ks, 2.0 ** -30)
    bed.upload()
    q = from_bits(to_bits(bed.rng.standard_normal((new, heads, dim)) * 1e9, dtype), dtype).reshape(new, heads * dim)
    padded = np.zeros((new, heads * dim + 24), np.float32)
    padded[:, :heads * dim] = q
    d = gpx.DeviceBuffer.from_numpy
    dq, out = d(to_bits(padded, dtype)), d(np.full((new, heads * dim + 8), 0x1234, np.uint16))
    gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, dtype, ctx, scale=0.011, q_ld=heads * dim + 24, out_ld=heads * dim + 8)
    gpx.device_sync()
    bits = out.download(np.uint16).reshape(new, -1)
    assert np.all(bits[:, heads * dim:] == 0x1234)
    got = from_bits(np.ascontiguousarray(bits[:, :heads * dim]), dtype).reshape(new, heads, dim)
    ref, _, weight = lm.attend(q.reshape(new, heads, dim), bed.k, bed.v, bed.ks, bed.vs, bed.table, [c], bed.first, float(np.float32(0.011)))
    check_attention(got, None, ref, None, weight, dtype, c, 448 * 2.0 ** 20 * 2.0 ** -24, 400)
    for b in (dq, out):
        b.free()
    bed.free()


def test_rows_that_one_key_dominates(gpx, ctx):
    """Scores hundreds apart: all but one probability vanish, and the running maximum jumps late."""
    c, heads, kv, dim, page = 700, 2, 1, 64, 64
    for at in (0, 333, 699):
        bed = Bed(gpx, [1], [c], heads, kv, dim, page, seed=11)
        q = np.zeros((1, heads, dim), np.float32)
        q[0, :, 0] = 8.0
        bed.k[..., 0] = 0
        bed.k[bed.table[0, at // page], 0, at % page, 0] = 0x7E  # 448
        bed.ks[:] = 1.0
        bed.upload()
        got, lse = run_attention(gpx, ctx, bed, q, "float16", heads)
        v = lm.decode(bed.v[bed.table[0, at // page], 0, at % page]) * bed.vs[bed.table[0, at // page], 0]
        assert np.array_equal(got[0, 0], v.astype(np.float16).astype(np.float32))
        assert abs(lse[0, 0] - 448) < 1e-3
        bed.free()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("power", [6, 24, 30, 60, 100])
def test_scores_of_any_magnitude(gpx, ctx, new, power):
    """One key ahead of all others by 2^power and more: it alone counts, whatever the rounding of such scores."""
    c, heads, kv, dim, page = 700, 2, 1, 128, 64
    q = np.zeros((new, heads, dim), np.float32)
    q[:, :, 0] = 2.0 ** power
    for at, scale in ((0, 1.0), (333, 0.75), (340, 1.0 / 3), (699, 1.3)):
        bed = Bed(gpx, [new], [c], heads, kv, dim, page, seed=at)
        bed.k[..., 0] = bed.rng.integers(0, 0x7D, bed.k[..., 0].shape)  # 384 at most
        bed.k[bed.table[0, at // page], 0, at % page, 0] = 0x7E  # 448
        bed.ks[:] = 1.0
        bed.upload()
        got, lse = run_attention(gpx, ctx, bed, q, "bfloat16", heads, causal=False, scale=scale)
        v = lm.decode(bed.v[bed.table[0, at // page], 0, at % page]) * bed.vs[bed.table[0, at // page], 0]
        assert np.array_equal(got, np.broadcast_to(from_bits(to_bits(v.astype(np.float32), "bfloat16"), "bfloat16"), got.shape))
        want = 448.0 * 2.0 ** power * float(np.float32(scale))
        assert np.all(np.abs(lse - want) <= 2.0 ** -20 * want)
        bed.free()


def test_cache_beyond_four_gigabytes(gpx, ctx):
    """Pages whose bytes lie past 32 bits; the pool is not initialised elsewhere."""
    pages, page, kv, dim, heads = 36000, 128, 8, 128, 16  # 4.7 GB of keys, as many of values
    small = Bed(gpx, [1, 2], [130, 300], heads, kv, dim, page, seed=2)
    far = pages - 1 - np.arange(small.pages)
    k, v = gpx.DeviceBuffer(pages * kv * page * dim), gpx.DeviceBuffer(pages * kv * page * dim)
    ks, vs = gpx.DeviceBuffer(pages * kv * 4), gpx.DeviceBuffer(pages * kv * 4)
    table = small.table.copy()
    for s, c in enumerate(small.context):
        for i in range(-(-int(c) // page)):
            table[s, i] = far[small.table[s, i]]
            for buf, src in ((k, small.k), (v, small.v)):
                buf.upload(src[small.table[s, i]], offset=int(far[small.table[s, i]]) * kv * page * dim)
            for buf, src in ((ks, small.ks), (vs, small.vs)):
                buf.upload(src[small.table[s, i]], offset=int(far[small.table[s, i]]) * kv * 4)
    small.upload()
    d = gpx.DeviceBuffer.from_numpy
    cache = gpx.KvCache(pages, page, kv, dim, k, v, ks, vs)
    dtable = d(table)
    batch = gpx.KvBatch(2, 3, 2, dtable, small.arrays[1], small.arrays[2], table.shape[1])
    bits = to_bits(small.rng.standard_normal((3, (heads + 2 * kv) * dim)), "bfloat16")
    dx = d(bits)
    width, at_k, at_v = bits.shape[1], 2 * heads * dim, 2 * (heads + kv) * dim
    outs = []
    for c, b in ((cache, batch), (small.cache, small.batch)):
        q, out = gpx.DeviceBuffer(3 * heads * dim * 2), gpx.DeviceBuffer(3 * heads * dim * 2)
        gpx.kv_append(c, b, dx, dx.ptr.value + at_k, dx.ptr.value + at_v, q, heads, "bfloat16", ctx, None, None, None, width, width, width)
        gpx.kv_attend(c, b, q, out, heads, "bfloat16", ctx)
        gpx.device_sync()
        outs.append(out.download(np.uint16))
        q.free(), out.free()
    assert np.array_equal(outs[0], outs[1])
    assert ctx.status() == (0, 0)
    cache.free(), small.free()
    for b in (k, v, ks, vs, dtable, dx):
        b.free()


# ---- scores -----------------------------------------------------------------------------------------

SCORES = [
    # rows, vocab, ld, dtype, top, temperature
    (1, 1, 1, "float32", 1, 1.0),
    (1, 7, 7, "bfloat16", 7, 1.0),
    (3, 31, 33, "float16", 5, 0.5),
    (2, 1000, 1001, "float32", 32, 1.3),
    (1, 30522, 30522, "float32", 5, 1.0),
    (5, 50257, 50257, "bfloat16", 20, 0.7),
    (7, 8191, 8195, "float16", 0, 1.0),
    (1300, 1025, 1025, "float16", 3, 1.0),
    (64, 4097, 4097, "bfloat16", 1, 2.0),
]


@pytest.mark.parametrize("case", SCORES, ids=lambda c: "%dx%d-%d-%s-%d-%g" % c)
def test_scores_match_the_definition(gpx, ctx, case):
    rows, vocab, ld, dtype, top, temperature = case
    rng = np.random.default_rng(rows + vocab)
    bits = to_bits(rng.standard_normal((rows, ld)) * 4, dtype)
    x = from_bits(bits, dtype)[:, :vocab]
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    if rows > 2:
        targets[0], targets[1] = -100, vocab
    check_scores(gpx, ctx, bits, x, targets, ld, dtype, top, temperature)


def check_scores(gpx, ctx, bits, x, targets, ld, dtype, top, temperature, offset=0):
    rows, vocab = x.shape
    d = gpx.DeviceBuffer.from_numpy
    dx, dt = d(bits), d(targets)
    outs = [gpx.DeviceBuffer(4 * rows) for _ in range(3)] + [gpx.DeviceBuffer(4 * rows * max(1, top)) for _ in range(2)]
    gpx.token_scores(dx.ptr.value + offset, rows, vocab, dtype, ctx, dt, *outs[:3], top, *outs[3:], temperature, ld)
    gpx.device_sync()
    lp, ent, lse = (b.download(np.float32, rows) for b in outs[:3])
    ids, top_lp = outs[3].download(np.int32, rows * top).reshape(rows, top), outs[4].download(np.float32, rows * top).reshape(rows, top)
    want = lm.scores(x, targets, top, 1.0 / temperature)
    assert np.array_equal(ids, want[3])
    with np.errstate(all="ignore"):
        size = np.abs(np.where(np.isfinite(x), x, 0)).max(1) / temperature
    # a logit is scaled and moved to base 2 (two roundings of its size), an exponential is good to 2^-21, sums of a row to 2^-20
    allowed = 2.0 ** -21 * (8 + size) + 2.0 ** -19
    for got, ref in ((lp, want[0]), (ent, want[1]), (lse, want[2])):
        fine = np.isfinite(ref)
        assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
        assert np.all(np.abs(got[fine] - ref[fine]) <= (2 * allowed * (1 + np.abs(ref) / 8))[fine]), np.max(np.abs(got[fine] - ref[fine]))
    fine = np.isfinite(want[4])
    assert np.array_equal(np.isnan(top_lp), np.isnan(want[4])) and np.array_equal(top_lp[np.isinf(want[4])], want[4][np.isinf(want[4])])
    bound = np.broadcast_to(allowed[:, None], fine.shape)
    assert np.all(np.abs(top_lp[fine] - want[4][fine]) <= 2 * bound[fine] * (1 + np.abs(want[4][fine]) / 8))
    for b in [dx, dt] + outs:
        b.free()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(6, 40), (6, 5003), (1500, 300)])
def test_scores_of_masked_tied_and_broken_rows(gpx, ctx, dtype, rows, vocab):
    rng = np.random.default_rng(vocab)
    x = np.round(rng.standard_normal((rows, vocab)) * 2).astype(np.float32)  # many ties
    lowest = -65504.0 if dtype == "float16" else -3.3e38
    x[0, rng.random(vocab) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2, rng.random(vocab) < 0.9] = lowest
    x[2, 3] = 0
    x[3, vocab // 2] = np.nan
    x[4, vocab - 1] = np.inf
    x[5] = lowest
    bits = to_bits(x, dtype)
    x = from_bits(bits, dtype)
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    targets[0] = int(np.flatnonzero(np.isneginf(x[0]))[0])  # a token that is masked
    targets[5] = vocab - 1
    check_scores(gpx, ctx, bits, x, targets, vocab, dtype, min(17, vocab), 1.0)


def test_scores_of_rows_off_any_boundary(gpx, ctx):
    bits = to_bits(np.random.default_rng(1).standard_normal(4 * 777 + 3), "bfloat16")
    for skip in (0, 1, 3):
        x = from_bits(bits[skip:skip + 3 * 777].reshape(3, 777), "bfloat16")
        check_scores(gpx, ctx, bits, x, np.arange(3, dtype=np.int32), 777, "bfloat16", 4, 1.0, offset=2 * skip)


# ---- what is refused, and what is reported -----------------------------------------------------------

def test_refusals(gpx, ctx):
    from gpreempt_b200 import binding as B

    bed = Bed(gpx, [1, 1], [20, 30], 4, 2, 64, 16).upload()
    x = gpx.DeviceBuffer(1 << 16)

    def refused(status, text, call, *args, **kw):
        with pytest.raises(gpx.GpxError) as e:
            call(*args, **kw)
        assert e.value.status == status and text in str(e.value), e.value

    def append(heads=4, dtype="bfloat16", q=x, k=x, v=x, q_out=x, rope=None, batch=bed.batch, **kw):
        gpx.kv_append(bed.cache, batch, q, k, v, q_out, heads, dtype, ctx, rope, **kw)

    def attend(heads=4, dtype="bfloat16", q=x, out=x, batch=bed.batch, **kw):
        gpx.kv_attend(bed.cache, batch, q, out, heads, dtype, ctx, **kw)

    odd = x.ptr.value + 2
    refused(B.OUT_OF_RANGE, "multiple of the cache's", append, heads=3)
    refused(B.OUT_OF_RANGE, "float32", append, dtype="float32")
    refused(B.FAIL, "NULL", append, k=None)
    refused(B.FAIL, "one of q and q_out", append, q_out=None)
    refused(B.FAIL, "aligned", append, v=odd)
    refused(B.FAIL, "multiples of 4", append, q_ld=4 * 64 + 2)
    refused(B.OUT_OF_RANGE, "longer", append, k_ld=64)
    refused(B.OUT_OF_RANGE, "rotated", append, rope=gpx.Rope(x, x, 40, 20))
    refused(B.OUT_OF_RANGE, "rotated", append, rope=gpx.Rope(x, x, 40, 72))
    refused(B.FAIL, "tables", append, rope=gpx.Rope(None, x, 40, 64))
    refused(B.FAIL, "tables", append, rope=gpx.Rope(x, x, 0, 64))
    refused(B.OUT_OF_RANGE, "multiple of the cache's", attend, heads=0)
    refused(B.OUT_OF_RANGE, "float64", attend, dtype="float64")
    refused(B.FAIL, "NULL", attend, out=None)
    refused(B.FAIL, "aligned", attend, q=odd)
    refused(B.OUT_OF_RANGE, "window", attend, window=-1)
    refused(B.OUT_OF_RANGE, "window", attend, window=3, causal=False)
    refused(B.OUT_OF_RANGE, "scale", attend, scale=-1.0)
    refused(B.OUT_OF_RANGE, "scale", attend, scale=float("nan"))
    refused(B.OUT_OF_RANGE, "longer", attend, out_ld=8)
    for seqs, tokens, most, ld, text in ((0, 2, 1, 2, "sequences"), (4097, 5000, 1, 2, "sequences"), (2, 2, 1, 0, "table_ld"), (2, 2, 3, 2, "new tokens")):
        batch = gpx.KvBatch(seqs, tokens, most, *bed.arrays, ld)
        refused(B.OUT_OF_RANGE, text, append, batch=batch)
        refused(B.OUT_OF_RANGE, text, attend, batch=batch)
    refused(B.FAIL, "NULL", attend, batch=gpx.KvBatch(2, 2, 1, bed.arrays[0], None, bed.arrays[2], 2))
    # nothing to do is no error
    gpx.kv_append(bed.cache, gpx.KvBatch(2, 0, 0, *bed.arrays, 2), None, x, x, None, 4, "bfloat16", ctx)
    gpx.kv_attend(bed.cache, gpx.KvBatch(2, 0, 0, *bed.arrays, 2), x, x, 4, "bfloat16", ctx)
    x.free(), bed.free()


@pytest.mark.parametrize("new", [1, 3])
def test_contradictions_on_the_device_are_reported_and_left_out(gpx, new):
    heads, kv, dim, page = 4, 2, 64, 16
    mine = gpx.LmContext()
    bed = Bed(gpx, [new] * 4, [40, 21, 33, 50], heads, kv, dim, page, seed=9).upload()
    d = gpx.DeviceBuffer.from_numpy
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), "bfloat16"), "bfloat16")
    ref, ref_lse, weight = lm.attend(q, bed.k, bed.v, bed.ks, bed.vs, bed.table, bed.context, bed.first)
    cos, sin = tables(45, dim)
    dcos, dsin = d(cos), d(sin)
    x = d(to_bits(bed.rng.standard_normal((bed.tokens, (heads + 2 * kv) * dim)), "bfloat16"))
    table, context, first = bed.table.copy(), bed.context.copy(), bed.first.copy()

    def upload(t=table, c=context, f=first):
        for a, b in zip(bed.arrays, (t, c, f)):
            a.upload(b)

    def append(rope=None):
        gpx.kv_append(bed.cache, bed.batch, None, x, x.ptr.value + 2 * kv * dim, None, heads, "bfloat16", mine, rope)
        gpx.device_sync()
        return mine.status()

    def others(left_out):
        got, lse = run_attention(gpx, mine, bed, q, "bfloat16", heads)
        keep = np.concatenate([np.arange(bed.first[s], bed.first[s + 1]) for s in range(4) if s != left_out])
        check_attention(got[keep], lse[keep], ref[keep], ref_lse[keep], weight[keep], "bfloat16", 50, 448 * 2.0 ** -5, 60)

    for value in (-1, bed.pages, 1 << 30):
        t = table.copy()
        t[2, 1 if new == 1 else 0] = value
        upload(t=t)
        others(2)
        assert mine.status() == (2, 2)
        mine.reset()
    t = table.copy()
    t[3, 3] = bed.pages  # the page of the new tokens
    upload(t=t)
    assert append() == (2, 3)
    mine.reset()
    bed.dk.upload(bed.k), bed.dv.upload(bed.v), bed.dks.upload(bed.ks), bed.dvs.upload(bed.vs)
    for value in (-5, 10000):
        c = context.copy()
        c[1] = value
        upload(c=c)
        others(1)
        assert mine.status() == (1, 1)
        mine.reset()
        assert append() == (1, 1)
        mine.reset()
        bed.dk.upload(bed.k), bed.dv.upload(bed.v), bed.dks.upload(bed.ks), bed.dvs.upload(bed.vs)
    f = first.copy()
    f[4] = bed.tokens + 1
    upload(f=f)
    others(3)
    assert mine.status() == (1, 3)
    mine.reset()
    upload()
    assert append(gpx.Rope(dcos, dsin, 45, dim)) == (3, 3)  # 50 tokens, 45 positions
    for b in (dcos, dsin, x):
        b.free()
    mine.free(), bed.free()


# ---- preemption -------------------------------------------------------------------------------------

def preempted_runs(gpx, launch, read, fresh, run_us, trials=6, at_least=2):
    """Raises the word at various moments of a launch, resumes until complete; results must be the same bits."""
    word = gpx.PreemptWord(1)
    blp = gpx.BlpContext(word, kernel_id=5)
    s = gpx.Stream(1)
    fresh()
    launch(blp, s)
    s.sync()
    assert blp.read()["stop_index"] == -1
    want = read()
    stopped = 0
    for trial in range(trials):
        fresh()
        blp.reset()
        word.clear()
        gpx.device_sync()
        for rounds in range(20):
            if trial == 0 and rounds == 0:
                word.raise_()
                gpx.device_sync()
            launch(blp, s)
            if rounds < 2:
                t0 = time.perf_counter()
                while (time.perf_counter() - t0) * 1e6 < run_us * trial / trials:
                    pass
                word.raise_()
            s.sync()
            word.clear()
            gpx.device_sync()
            st = blp.read()
            if st["stop_index"] == -1:
                break
            assert st["stop_index"] == 5
            if trial == 0 and rounds == 0:
                assert st["cursor"] == 0 and st["tiles_run"] == 0
            stopped += 1
            blp.rearm()
        else:
            raise AssertionError("not complete after 20 launches")
        for a, b in zip(read(), want):
            assert np.array_equal(a, b)
    assert stopped >= at_least
    for o in (blp, word, s):
        (o.free if hasattr(o, "free") else o.destroy)()
    return want


def test_attention_drains_and_resumes_bit_identically(gpx, ctx):
    new, context, heads, kv, dim, page = [1] * 40, [8000 + 37 * i for i in range(40)], 16, 4, 128, 64
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=4).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), "bfloat16"), "bfloat16")
    dq = gpx.DeviceBuffer.from_numpy(to_bits(q, "bfloat16"))
    out = gpx.DeviceBuffer(bed.tokens * heads * dim * 2)
    want = preempted_runs(gpx, lambda blp, s: gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, "bfloat16", ctx, blp=blp, stream=s),
                          lambda: [out.download(np.uint16)], out.zero, 150)
    some = slice(0, 3)
    ref, _, weight = lm.attend(q[some], bed.k, bed.v, bed.ks, bed.vs, bed.table, context[some], bed.first[:4])
    got = from_bits(want[0], "bfloat16").reshape(bed.tokens, heads, dim)[some]
    check_attention(got, None, ref, None, weight, "bfloat16", max(context), 448 * 2.0 ** -5, 60)
    dq.free(), out.free(), bed.free()


def test_prompt_attention_drains_and_resumes_bit_identically(gpx, ctx):
    new, context, heads, kv, dim, page = [700, 900], [3000, 900], 16, 4, 128, 64
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=4).upload()
    q = from_bits(to_bits(bed.rng.standard_normal((bed.tokens, heads, dim)), "bfloat16"), "bfloat16")
    dq = gpx.DeviceBuffer.from_numpy(to_bits(q, "bfloat16"))
    out = gpx.DeviceBuffer(bed.tokens * heads * dim * 2)
    preempted_runs(gpx, lambda blp, s: gpx.kv_attend(bed.cache, bed.batch, dq, out, heads, "bfloat16", ctx, blp=blp, stream=s),
                   lambda: [out.download(np.uint16)], out.zero, 200)
    dq.free(), out.free(), bed.free()


def test_append_drains_and_resumes_bit_identically(gpx, ctx):
    new, context, heads, kv, dim, page = [3000, 2500, 4000], [3010, 2600, 4000], 8, 8, 128, 64
    bed = Bed(gpx, new, context, heads, kv, dim, page, seed=6).upload()
    x = gpx.DeviceBuffer.from_numpy(to_bits(bed.rng.standard_normal((bed.tokens, 3 * heads * dim)), "bfloat16"))
    q, width = gpx.DeviceBuffer(bed.tokens * heads * dim * 2), 3 * heads * dim
    cos, sin = tables(4001, dim)
    dcos, dsin = gpx.DeviceBuffer.from_numpy(cos), gpx.DeviceBuffer.from_numpy(sin)
    rope = gpx.Rope(dcos, dsin, 4001, dim)

    def fresh():
        q.zero()
        for b, a in ((bed.dk, bed.k), (bed.dv, bed.v), (bed.dks, bed.ks), (bed.dvs, bed.vs)):
            b.upload(a)

    at = x.ptr.value
    preempted_runs(gpx, lambda blp, s: gpx.kv_append(bed.cache, bed.batch, at, at + 2 * heads * dim, at + 4 * heads * dim, q, heads, "bfloat16",
                                                     ctx, rope, blp, s, width, width, width),
                   lambda: [q.download(np.uint16), *bed.download()], fresh, 60)
    for b in (x, q, dcos, dsin):
        b.free()
    bed.free()


@pytest.mark.parametrize("rows", [37, 3000])
def test_scores_drain_and_resume_bit_identically(gpx, ctx, rows):
    vocab = 40001
    x = gpx.DeviceBuffer(rows * vocab * 2)
    gpx.fill_uniform(x, rows * vocab, True, 3, lo=-9.0, hi=9.0)
    outs = [gpx.DeviceBuffer(4 * rows) for _ in range(2)] + [gpx.DeviceBuffer(40 * rows) for _ in range(2)]

    def launch(blp, s):
        gpx.token_scores(x, rows, vocab, "bfloat16", ctx, entropy=outs[0], lse=outs[1], top=10, top_ids=outs[2], top_logprob=outs[3], blp=blp, stream=s)

    preempted_runs(gpx, launch, lambda: [b.download(np.uint32) for b in outs], lambda: [b.zero() for b in outs], 10 if rows == 37 else 80,
                   at_least=1 if rows == 37 else 2)  # (the few rows take a few microseconds)
    for b in [x] + outs:
        b.free()
