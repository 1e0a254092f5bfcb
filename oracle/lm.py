"""Restatement of the decoder's serving step in 64 bits (numpy): paged 8-bit cache, attention over it, token scores."""
from __future__ import annotations

import numpy as np

# ---- OCP e4m3: sign, four bits of exponent (bias 7), three of mantissa; 0x7f is NaN, there is no infinity ------------

_code = np.arange(256)
_exp, _man = (_code >> 3) & 15, _code & 7
E4M3 = np.where(_exp == 0, _man * 2.0 ** -9, (8 + _man) * 2.0 ** (_exp - 10.0))
E4M3 = np.where(_code & 0x80, -E4M3, E4M3)
E4M3[[0x7F, 0xFF]] = np.nan
_FINITE = E4M3[:127]  # codes 0 .. 126, ascending
_BETWEEN = (_FINITE[1:] + _FINITE[:-1]) / 2


def decode(codes: np.ndarray) -> np.ndarray:
    return E4M3[codes]


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code, ties to the even one; what is not finite becomes NaN."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    low, high = np.searchsorted(_BETWEEN, a, "left"), np.searchsorted(_BETWEEN, a, "right")
    code = np.where(low == high, low, np.where(low % 2 == 0, low, high))
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isfinite(x), code, 0x7F).astype(np.uint8)


def block_scale(x: np.ndarray) -> np.ndarray:
    """Smallest power of two with which the largest finite magnitude is at most 448, of each head of x [token][head][element]."""
    amax = np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=(0, 2)).astype(np.float64)
    m, e = np.frexp(amax / 448.0)  # amax / 448 = m 2^e, 1/2 <= m < 1
    e = np.where(amax == 0, -126, np.where(m == 0.5, e - 1, e))
    return np.ldexp(1.0, np.maximum(e, -126).astype(int)).astype(np.float32)


def turn(x: np.ndarray, positions: np.ndarray, cos: np.ndarray, sin: np.ndarray, rotated: int, paired: bool) -> np.ndarray:
    """Rotation as the operator defines it: float, each product and sum rounded.  x [token][head][element]."""
    x = x.astype(np.float32).copy()
    if not rotated:
        return x
    c, s = cos[positions][:, None, :].astype(np.float32), sin[positions][:, None, :].astype(np.float32)
    a_at, b_at = (slice(0, rotated, 2), slice(1, rotated, 2)) if paired else (slice(0, rotated // 2), slice(rotated // 2, rotated))
    a, b = x[..., a_at].copy(), x[..., b_at].copy()
    with np.errstate(all="ignore"):
        x[..., a_at] = a * c - b * s
        x[..., b_at] = b * c + a * s
    return x


def append(k_codes, v_codes, k_scale, v_scale, table, context, first, k, v, cos=None, sin=None, rotated=0, paired=False):
    """Appends keys and values [token][kv_head][element] in place."""
    page_tokens = k_codes.shape[2]
    for s in range(len(context)):
        n = first[s + 1] - first[s]
        pos = np.arange(context[s] - n, context[s])
        rows = slice(first[s], first[s + 1])
        for codes, scales, x in ((k_codes, k_scale, turn(k[rows], pos, cos, sin, rotated, paired)), (v_codes, v_scale, v[rows].astype(np.float32))):
            done = 0
            while done < n:
                begin = pos[done] % page_tokens
                count = min(page_tokens - begin, n - done)
                page = table[s][pos[done] // page_tokens]
                new = x[done:done + count]
                scale = block_scale(new)
                if begin:
                    old = scales[page].copy()
                    scale = np.maximum(scale, old)
                    held = decode(codes[page, :, :begin]) * (old / scale)[:, None, None].astype(np.float64)
                    codes[page, :, :begin] = np.where((old < scale)[:, None, None], encode(held), codes[page, :, :begin])
                scales[page] = scale
                codes[page, :, begin:begin + count] = encode(new.astype(np.float64) / scale[None, :, None]).transpose(1, 0, 2)
                done += count


def attend(q, k_codes, v_codes, k_scale, v_scale, table, context, first, scale=None, causal=True, window=0):
    """Returns out, lse and sum |p v| (for error bounds), in 64 bits; q [token][head][element]."""
    tokens, heads, dim = q.shape
    page_tokens, kv_heads = k_codes.shape[2], k_codes.shape[1]
    scale = scale if scale else 1.0 / np.sqrt(dim)
    out, weight = np.zeros((tokens, heads, dim)), np.zeros((tokens, heads, dim))
    lse = np.full((tokens, heads), -np.inf)
    group = heads // kv_heads
    for s in range(len(context)):
        n, c = first[s + 1] - first[s], context[s]
        pages = table[s][: -(-c // page_tokens)]
        if n == 0 or c == 0:
            continue
        k = (decode(k_codes[pages]) * k_scale[pages][:, :, None, None].astype(np.float64)).transpose(1, 0, 2, 3).reshape(kv_heads, -1, dim)
        v = (decode(v_codes[pages]) * v_scale[pages][:, :, None, None].astype(np.float64)).transpose(1, 0, 2, 3).reshape(kv_heads, -1, dim)
        for i in range(n):
            high = min(c, max(0, c - n + i + 1)) if causal else c
            low = max(0, c - n + i + 1 - window) if window else 0
            if high <= low:
                continue
            for h in range(heads):
                with np.errstate(all="ignore"):
                    x = k[h // group, low:high] @ q[first[s] + i, h].astype(np.float64) * scale
                    top = x.max()
                    p = np.exp(x - top)
                    total = p.sum()
                    p = p / total
                    out[first[s] + i, h] = p @ v[h // group, low:high]
                    weight[first[s] + i, h] = p @ np.abs(np.nan_to_num(v[h // group, low:high]))
                    lse[first[s] + i, h] = top + np.log(total)
    return out, lse, weight


def scores(logits, targets=None, top=0, inv_temperature=1.0):
    """logprob, entropy, lse, top_ids, top_logprob of rows of logits, in 64 bits.  The order of alternatives is that of
    the logits times the temperature in float, lowest index first among equals and NaN before everything."""
    x32 = (logits.astype(np.float32) * np.float32(inv_temperature)).astype(np.float32)
    x = x32.astype(np.float64)
    with np.errstate(all="ignore"):
        top_x = x.max(1, keepdims=True)
        e = np.exp(x - np.where(np.isneginf(top_x), 0.0, top_x))
        total = e.sum(1, keepdims=True)
        lse = (np.where(np.isneginf(top_x), 0.0, top_x) + np.log(total))[:, 0]
        y = x - lse[:, None]
        p = e / total
        entropy = -np.where(p == 0, 0.0, p * y).sum(1)
        logprob = None
        if targets is not None:
            picked = np.take_along_axis(y, np.clip(targets, 0, x.shape[1] - 1)[:, None], 1)[:, 0]
            logprob = np.where(targets < 0, 0.0, np.where(targets >= x.shape[1], np.nan, picked))
        rank = np.where(np.isnan(x32), np.inf, x32)
        order = np.stack([np.lexsort((np.arange(x.shape[1]), -r, ~np.isnan(v))) for r, v in zip(rank, x32)])[:, :top]
        return logprob, entropy, lse, order, np.take_along_axis(y, order, 1)
