"""The operators of a decoder's serving step, as cases that can be timed and compared.

  append   new keys and values go into a paged cache of 8-bit codes with a scale for each page and head; the position
           rotation is applied to queries and keys on the way
  attend   attention of the new tokens over such a cache: single tokens, a few, prompt chunks, or an encoder's states
  scores   log probabilities of given tokens, entropies and the top alternatives, from logits

Every case exists in a plain form (elementary torch operations in 32 bits) and as calls of the framework.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # One token of one conversation goes into its cache: launch latency.
        _append("append-1x1", 1, 1, 128, 32, 8, 128, 64, "bfloat16"),
        # A decoding batch with small pages, as many heads of keys as of queries, adjacent elements rotated.
        _append("append-64x1", 64, 1, 4000, 12, 12, 64, 16, "float16", paired=True),
        # Prompts of uneven lengths are taken in at once.
        _append("append-prompts", 8, 4096, 300, 32, 8, 128, 64, "bfloat16"),
        # One token of one conversation of a few hundred: latency.
        _attend("attend-1x1-517", 1, 1, 516, 32, 8, 128, 64, "bfloat16"),
        # One token over a very long conversation: the keys are the only long axis.
        _attend("attend-1x1-131071", 1, 1, 131070, 32, 8, 128, 128, "bfloat16"),
        # A decoding batch of uneven conversations, the common load of a server.
        _attend("attend-64x1-16384", 64, 1, 16383, 32, 8, 128, 64, "bfloat16"),
        # A few proposed tokens a conversation are checked at once; heads of 64 without groups.
        _attend("attend-16x5-2000", 16, 5, 1995, 12, 12, 64, 32, "float16"),
        # Chunks of two long prompts behind what was taken in before.
        _attend("attend-2x2048-8192", 2, 2048, 6144, 32, 8, 128, 64, "bfloat16"),
        # Decoder tokens over an encoder's 512 states: no causal mask.
        _attend("attend-cross-8x37-512", 8, 37, 512, 12, 12, 64, 64, "float16", causal=False),
        # The next-token distribution of one row of an odd vocabulary.
        _scores("scores-1x30522", 1, 30522, 30522, "float32", 5, 1.0),
        # A decoding batch with a temperature and twenty alternatives.
        _scores("scores-64x131072", 64, 131072, 131072, "bfloat16", 20, 0.7),
        # A prompt is scored token by token; rows are padded, the vocabulary is odd.
        _scores("scores-4096x50257", 4096, 50257, 50264, "float16", 1, 1.0),
    ]


def _append(name, seqs, new, past, heads, kv_heads, dim, page, dtype, paired=False, rotated=0):
    return {"name": name, "kind": "append", "seqs": seqs, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "paired": paired, "rotated": rotated or dim}


def _attend(name, seqs, new, past, heads, kv_heads, dim, page, dtype, causal=True, window=0):
    return {"name": name, "kind": "attend", "seqs": seqs, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "causal": causal, "window": window}


def _scores(name, rows, vocab, ld, dtype, top, temperature):
    return {"name": name, "kind": "scores", "rows": rows, "vocab": vocab, "ld": ld, "dtype": dtype, "top": top, "temperature": temperature}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(32, 8), (12, 12), (16, 1), (28, 4), (40, 8), (8, 2), (64, 8), (6, 6), (24, 2)]


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "scores"])
    if kind == "scores":
        vocab = _log_int(rng, 1000, 200000)
        rows = _log_int(rng, 1, min(4096, (1 << 27) // vocab))
        case = _scores("", rows, vocab, vocab + rng.choice([0, 0, 1, 7, 64]), rng.choice(sorted(DTYPES)), rng.randint(0, 20),
                       rng.choice([1.0, 0.7, 1.3]))
    else:
        heads, kv_heads = rng.choice(HEADS)
        dim, page, dtype = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["bfloat16", "float16"])
        seqs = _log_int(rng, 1, 128)
        if kind == "append":
            new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(4096, 16384 // seqs)))
            case = _append("", seqs, new, _log_int(rng, 1, 8192), heads, kv_heads, dim, page, dtype, rng.random() < 0.5,
                           rng.choice([dim, dim, dim // 2]))
        else:
            form = rng.choice(["one", "one", "few", "chunk", "cross"])
            if form == "chunk":
                seqs = min(seqs, 16)
            new = {"one": 1, "few": rng.randint(2, 8), "chunk": _log_int(rng, 9, 2048 // seqs), "cross": _log_int(rng, 1, 64)}[form]
            # (what the plain form lays out: decoded keys, and scores)
            most = min(16384, (1 << 28) // (seqs * kv_heads * dim), (1 << 29) // (seqs * heads * new))
            past = max(1, _log_int(rng, 1, max(1, most - new)))
            case = _attend("", seqs, new, past, heads, kv_heads, dim, page, dtype, form != "cross",
                           rng.choice([0, 0, _log_int(rng, 1, 4096)]) if form != "cross" else 0)
    del case["name"]
    return case


def _spread(count, most, least, step):
    """`count` uneven lengths from `least` to `most`, the first of them `most`."""
    return [most - int((most - least) * ((i * step) % 1.0)) for i in range(count)]


def _lengths(case):
    """New tokens and tokens in all of every sequence."""
    if case["kind"] == "attend" and not case["causal"]:  # the states of an encoder: none of them is a new token's
        new = _spread(case["seqs"], case["new"], max(1, case["new"] // 4), 0.7548776662)
        return new, _spread(case["seqs"], case["past"], max(1, case["past"] // 8), 0.6180339887)
    new = _spread(case["seqs"], case["new"], max(1, case["new"] // 4), 0.7548776662)
    past = _spread(case["seqs"], case["past"], case["past"] // 16, 0.6180339887)
    return new, [n + p for n, p in zip(new, past)]


# ---- what a user's program has in hand -------------------------------------------------------------

_kept = {}


def _context():
    """The scratch memory a process keeps for these operators."""
    if "context" not in _kept:
        from gpreempt_b200 import api

        api.init_cuda(0)
        _kept["context"] = api.LmContext()
    return _kept["context"]


def _cache(case, context, g):
    """A pool of pages in no particular order with finite codes everywhere, as recycled pages have, and the pages' scales."""
    page, kv, dim, seqs = case["page"], case["kv_heads"], case["dim"], case["seqs"]
    per_seq = [-(-c // page) for c in context]
    pages = sum(per_seq) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(per_seq)
    table = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(per_seq):
        table[s, :n] = order[at:at + n]
        at += n

    def codes(spread):
        # values of unit size, some heads larger than others; codes use the range that their block's scale gives them
        x = torch.empty(pages, kv, page, dim, dtype=torch.uint8, device="cuda")
        scale = torch.empty(pages, kv, dtype=torch.float32, device="cuda")
        some = max(1, (1 << 28) // (kv * page * dim))
        head = torch.exp(torch.randn(kv, generator=g, device="cuda") * spread)
        for p in range(0, pages, some):
            y = torch.randn(min(some, pages - p), kv, page, dim, generator=g, device="cuda") * head[:, None, None]
            top = torch.exp2(torch.ceil(torch.log2(y.abs().amax((2, 3)) / E4M3_MAX)))
            scale[p:p + some] = top
            x[p:p + some] = (y / top[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        return x, scale

    k, k_scale = codes(0.3)
    v, v_scale = codes(0.5)
    return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "table": table}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "scores":
        rows, vocab, ld = case["rows"], case["vocab"], case["ld"]
        s["logits"] = torch.empty(rows, ld, dtype=dtype, device="cuda")
        some = max(1, (1 << 27) // ld)
        for r in range(0, rows, some):
            # a broad background and a few hundred likely tokens a row
            x = torch.randn(min(some, rows - r), ld, generator=g, device="cuda") * 2.0
            likely = torch.randint(0, vocab, (x.shape[0], 256), generator=g, device="cuda")
            x.scatter_add_(1, likely, torch.rand(likely.shape, generator=g, device="cuda") * 12.0)
            s["logits"][r:r + some] = x.to(dtype)
        s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
        if own:
            f32, top = {"dtype": torch.float32, "device": "cuda"}, case["top"]
            s["out"] = {"logprob": torch.empty(rows, **f32), "entropy": torch.empty(rows, **f32), "top_logprob": torch.empty(rows, top, **f32),
                        "top_ids": torch.empty(rows, top, dtype=torch.int32, device="cuda")}
            s["context"] = _context()
        return s

    new, context = _lengths(case)
    heads, kv, dim, seqs, tokens = case["heads"], case["kv_heads"], case["dim"], case["seqs"], sum(new)
    s.update(_cache(case, context, g))
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(context, dtype=torch.int32, device="cuda")
    s["tokens"] = tokens
    if case["kind"] == "append":
        # one projection's output holds queries, keys and values of a token side by side
        packed = torch.empty(tokens, (heads + 2 * kv) * dim, dtype=dtype, device="cuda")
        packed.normal_(generator=g)
        s["packed"] = packed
        s["q"], s["k_new"], s["v_new"] = packed[:, :heads * dim], packed[:, heads * dim:(heads + kv) * dim], packed[:, (heads + kv) * dim:]
        half = case["rotated"] // 2
        angle = torch.arange(max(context), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = torch.empty(tokens, heads * dim, dtype=dtype, device="cuda").normal_(generator=g)
        s["q"] *= 1.5
    if own:
        from gpreempt_b200 import api

        s["context"] = _context()
        s["out"] = torch.empty(tokens, heads * dim, dtype=dtype, device="cuda")
        s["lse"] = torch.empty(tokens, heads, dtype=torch.float32, device="cuda")
        s["cache"] = api.KvCache(s["k"].shape[0], case["page"], kv, dim, s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = api.KvBatch(seqs, tokens, max(new), s["table"], s["lengths"], s["first"], s["table"].shape[1])
        if case["kind"] == "append":
            s["rope"] = api.Rope(s["cos"], s["sin"], s["cos"].shape[0], case["rotated"], case["paired"])
    return s


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "append":
        return _append_own(state) if own else _append_plain(state)
    if kind == "attend":
        return _attend_own(state) if own else _attend_plain(state)
    return _scores_own(state) if own else _scores_plain(state)


def _append_own(s):
    from gpreempt_b200 import api

    case = s["case"]
    ld = s["packed"].shape[1]
    api.kv_append(s["cache"], s["batch"], s["q"], s["k_new"], s["v_new"], s["out"], case["heads"], case["dtype"], s["context"],
                  rope=s["rope"], q_ld=ld, k_ld=ld, v_ld=ld)
    f8 = torch.float8_e4m3fn
    return {"q": s["out"], "k": s["k"].view(f8), "v": s["v"].view(f8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attend_own(s):
    from gpreempt_b200 import api

    case = s["case"]
    api.kv_attend(s["cache"], s["batch"], s["q"], s["out"], case["heads"], case["dtype"], s["context"], causal=case["causal"],
                  window=case["window"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _scores_own(s):
    from gpreempt_b200 import api

    case, out = s["case"], s["out"]
    api.token_scores(s["logits"], case["rows"], case["vocab"], case["dtype"], s["context"], targets=s["targets"], logprob=out["logprob"],
                     entropy=out["entropy"], top=case["top"], top_ids=out["top_ids"], top_logprob=out["top_logprob"],
                     temperature=case["temperature"], ld=case["ld"])
    return out


def _places(s):
    """Sequence and position of every new token."""
    first = s["first"].long()
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(first[1:].contiguous(), token, right=True)
    new = first[1:] - first[:-1]
    return seq, token - first[seq], (s["lengths"].long() - new)[seq] + token - first[seq]


def _append_plain(s):
    case = s["case"]
    page, dim, rot = case["page"], case["dim"], case["rotated"]
    seq, _, pos = _places(s)
    at = s["table"].long()[seq, pos // page]
    slot = pos % page
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]

    def rotate(x):
        x = x.float().reshape(x.shape[0], -1, dim)
        r, rest = x[..., :rot], x[..., rot:]
        if case["paired"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, rest], -1)

    # the only page of a sequence that may hold tokens already is the one its first new token goes to
    past = s["lengths"].long() - (s["first"][1:] - s["first"][:-1]).long()
    begun = s["table"].long().gather(1, (past // page).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0]
    has = past % page

    def store(codes, scale, x):
        amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        bits = amax.view(torch.int32)
        want = ((((bits + 0x1fffff) >> 23) - 8).clamp(min=1) << 23).view(torch.float32)  # the power of two at or above amax / 448
        old = scale[begun]
        fresh = torch.zeros_like(scale).index_reduce_(0, at, want, "amax")
        fresh[begun] = torch.maximum(fresh[begun], torch.where(has[:, None] > 0, old, 0.0))
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
        touched[at] = True
        scale.copy_(torch.where(touched[:, None], fresh, scale))
        kept = codes[begun]
        again = (kept.view(torch.float8_e4m3fn).float() * (old / scale[begun])[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        held = torch.arange(page, device="cuda")[None, :] < has[:, None]
        codes[begun] = torch.where(held[:, None, :, None], again, kept)
        codes[at, :, slot] = (x / scale[at][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)

    q = rotate(s["q"]).reshape(s["tokens"], -1).to(DTYPES[case["dtype"]])
    store(s["k"], s["k_scale"], rotate(s["k_new"]))
    store(s["v"], s["v_scale"], s["v_new"].float().reshape(s["tokens"], -1, dim))
    f8 = torch.float8_e4m3fn
    return {"q": q, "k": s["k"].view(f8), "v": s["v"].view(f8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attend_plain(s):
    case = s["case"]
    heads, kv, dim, seqs, page = case["heads"], case["kv_heads"], case["dim"], case["seqs"], case["page"]
    group = heads // kv
    seq, i, pos = _places(s)
    table = s["table"].long()

    def decoded(codes, scale):
        x = codes[table].view(torch.float8_e4m3fn).float() * scale[table][:, :, :, None, None]
        return x.transpose(1, 2).reshape(seqs, kv, -1, dim)

    k, v = decoded(s["k"], s["k_scale"]), decoded(s["v"], s["v_scale"])
    most = case["new"]
    q = torch.zeros(seqs, most, heads, dim, device="cuda")
    q[seq, i] = s["q"].float().reshape(-1, heads, dim)
    where = torch.full((seqs, most), -1, dtype=torch.int64, device="cuda")
    where[seq, i] = pos
    q = q.reshape(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(dim)).reshape(seqs, kv, group, most, -1)
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key[None, :] < s["lengths"][:, None])[:, None, :].expand(-1, most, -1)
    if case["causal"]:
        seen = seen & (key[None, None, :] <= where[:, :, None])
    if case["window"]:
        seen = seen & (key[None, None, :] > where[:, :, None] - case["window"])
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top)[..., 0]
    o = (p.reshape(seqs, kv, group * most, -1) @ v).reshape(seqs, kv, group, most, dim) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * dim)[seq, i]
    return {"out": o.to(DTYPES[case["dtype"]]), "lse": lse.permute(0, 3, 1, 2).reshape(seqs, most, heads)[seq, i]}


def _scores_plain(s):
    case = s["case"]
    x = s["logits"][:, :case["vocab"]].float() * (1.0 / case["temperature"])
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    lse = m + total.log()
    logprob = x.gather(1, s["targets"].long()[:, None]) - lse
    entropy = total.log() - torch.where(e > 0, (x - m) * e, 0.0).sum(1, keepdim=True) / total
    top, ids = x.sort(dim=1, descending=True, stable=True)
    return {"logprob": logprob[:, 0], "entropy": entropy[:, 0], "top_logprob": top[:, :case["top"]] - lse,
            "top_ids": ids[:, :case["top"]].to(torch.int32)}


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["kind"] == "scores":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * (4 if case["dtype"] == "float32" else 2) + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * cells}
    new, context = _lengths(case)
    heads, kv, dim, page, tokens = case["heads"], case["kv_heads"], case["dim"], case["page"], sum(new)
    if case["kind"] == "append":
        # read: queries, keys, values, a row of the tables a token; written: queries, codes; a scale of both a page and head
        pages = sum(-(-c // page) - (c - n) // page for n, c in zip(new, context))
        moved = 2 * tokens * (heads + 2 * kv) * dim + 4 * tokens * case["rotated"] + 2 * tokens * heads * dim + 2 * tokens * kv * dim
        return {"bytes": moved + 16 * pages * kv + 4 * pages, "flops": 4 * tokens * (heads + 2 * kv) * dim}
    moved = pairs = 0
    for n, c in zip(new, context):
        low = 0
        if case["causal"]:
            # row i sees the keys up to its own position, at most `window` of them
            rows = [c - n + i + 1 for i in range(n)]
            if case["window"]:
                low = max(0, c - n + 1 - case["window"])
                rows = [min(r, case["window"]) for r in rows]
            pairs += sum(rows)
        else:
            pairs += n * c
        moved += (c - low) * kv * dim * 2 + (-(-c // page) - low // page) * (8 * kv + 4)
    return {"bytes": moved + 4 * tokens * heads * dim + 4 * tokens * heads, "flops": 4 * pairs * heads * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "scores":
        return _exact_scores(s)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(s)


def _exact_scores(s):
    case = s["case"]
    rows, top = case["rows"], case["top"]
    logprob, entropy = torch.empty(rows, dtype=torch.float64), torch.empty(rows, dtype=torch.float64)
    best = torch.empty(rows, top, dtype=torch.float64)
    some = max(1, (1 << 26) // case["vocab"])
    for r in range(0, rows, some):
        x = s["logits"][r:r + some, :case["vocab"]].double() / case["temperature"]
        lse = torch.logsumexp(x, 1)
        logprob[r:r + some] = (x.gather(1, s["targets"][r:r + some].long()[:, None])[:, 0] - lse).cpu()
        y = x - lse[:, None]
        entropy[r:r + some] = -torch.special.xlogy(y.exp(), y.exp()).sum(1).cpu()
        best[r:r + some] = torch.topk(y, top, 1).values.cpu()
    return {"logprob": logprob, "entropy": entropy, "top_logprob": best, "top_ids": None}


def _exact_append(s):
    """Codes are what the stored numbers stand for before they are rounded to 8 bits."""
    case = s["case"]
    page, dim, rot, heads, kv = case["page"], case["dim"], case["rotated"], case["heads"], case["kv_heads"]
    new, context = _lengths(case)
    half = rot // 2
    k = s["k"].view(torch.float8_e4m3fn).double()
    v = s["v"].view(torch.float8_e4m3fn).double()
    k_scale, v_scale = s["k_scale"].double(), s["v_scale"].double()
    q = torch.empty(s["tokens"], heads * dim, dtype=torch.float64, device="cuda")
    # element j of a head is turned against its partner by the angle of their pair
    j = torch.arange(rot, device="cuda")
    pair = j // 2 if case["paired"] else j % half
    partner = j ^ 1 if case["paired"] else (j + half) % rot
    sign = torch.where(j % 2 == 0 if case["paired"] else j < half, -1.0, 1.0).double()

    def turned(x, where):
        x = x.double().reshape(x.shape[0], -1, dim)
        c, t = s["cos"].double()[where][:, pair], s["sin"].double()[where][:, pair]
        y = x.clone()
        y[..., :rot] = x[..., :rot] * c[:, None] + sign * t[:, None] * x[..., partner]
        return y

    def block(codes, scale, p, begin, x):
        """Tokens x [n][heads][dim] go to the slots from `begin` of page p."""
        amax = x.abs().amax((0, 2))
        want = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(min=-126))
        if begin:
            want = torch.maximum(want, scale[p])
            codes[p, :, :begin] *= (scale[p] / want)[:, None, None]
        scale[p] = want
        codes[p, :, begin:begin + x.shape[0]] = (x / want[None, :, None]).transpose(0, 1)

    at = 0
    tables = s["table"].tolist()
    for i, (n, c) in enumerate(zip(new, context)):
        where = torch.arange(c - n, c, device="cuda")
        q[at:at + n] = turned(s["q"][at:at + n], where).reshape(n, -1)
        ks, vs = turned(s["k_new"][at:at + n], where), s["v_new"][at:at + n].double().reshape(n, kv, dim)
        done = 0
        while done < n:
            begin = (c - n + done) % page
            some = min(page - begin, n - done)
            p = tables[i][(c - n + done) // page]
            block(k, k_scale, p, begin, ks[done:done + some])
            block(v, v_scale, p, begin, vs[done:done + some])
            done += some
        at += n
    return {"q": q, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


def _exact_attend(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    new, context = _lengths(case)
    out = torch.zeros(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], heads), float("-inf"), dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, c) in enumerate(zip(new, context)):
        pages = s["table"][i, :-(-c // case["page"])].long()
        for h in range(heads):
            of = h // (heads // kv)
            k = (s["k"][pages, of].view(torch.float8_e4m3fn).double() * s["k_scale"][pages, of].double()[:, None, None]).reshape(-1, dim)[:c]
            v = (s["v"][pages, of].view(torch.float8_e4m3fn).double() * s["v_scale"][pages, of].double()[:, None, None]).reshape(-1, dim)[:c]
            x = s["q"][at:at + n, h * dim:(h + 1) * dim].double() @ k.T / math.sqrt(dim)
            if case["causal"]:
                key, row = torch.arange(c, device="cuda")[None], torch.arange(c - n, c, device="cuda")[:, None]
                hidden = key > row
                if case["window"]:
                    hidden |= key <= row - case["window"]
                x.masked_fill_(hidden, float("-inf"))
            lse[at:at + n, h] = torch.logsumexp(x, 1)
            out[at:at + n, h] = torch.softmax(x, 1) @ v
        at += n
    return {"out": out.reshape(s["tokens"], -1), "lse": lse}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(12)]:
        print(c, work(c))
