"""The 8-bit paged cache in 64 bits (numpy): what tests compare the kernels
with.  Written from the definitions in include/dsd_hip.h."""
from __future__ import annotations

import numpy as np

E4M3, INT8 = 0, 1
LARGEST = {E4M3: 448.0, INT8: 127.0}
TINY = np.float32(2.0 ** -126)


def e4m3_table():
    code = np.arange(256)
    exponent, fraction = (code >> 3) & 15, code & 7
    size = np.where(exponent == 0, fraction * 2.0 ** -9, (8 + fraction) * 2.0 ** (exponent - 10.0))
    size = np.where(code & 127 == 127, np.nan, size)
    return np.where(code >= 128, -size, size)


_TABLE = e4m3_table()


def numbers(fmt, codes):
    """The numbers that uint8 codes stand for."""
    if fmt == INT8:
        return codes.view(np.int8).astype(np.float64)
    return _TABLE[codes]


def nearest(fmt, x):
    """The number of the format next to x, halves to the even code."""
    if fmt == INT8:
        return np.clip(np.rint(np.where(np.isnan(x), 0.0, x)), -127, 127)
    x = np.clip(x, -448.0, 448.0)
    with np.errstate(all="ignore"):
        exponent = np.frexp(np.where(np.isnan(x), 0.0, x))[1] - 1
    step = np.exp2(np.maximum(exponent, -6) - 3.0)
    return np.rint(x / step) * step


def scale_for(fmt, most):
    most = np.asarray(most, np.float64).astype(np.float32)
    if fmt == INT8:
        return np.maximum((most.astype(np.float64) / 127).astype(np.float32), TINY)
    fraction, exponent = np.frexp(most)
    power = np.where(most > 0, exponent - 9 + (fraction > 0.875), -126)
    return np.exp2(np.maximum(power, -126).astype(np.float64)).astype(np.float32)


def rotate(x, positions, inv_freq, interleaved=False, magnitude=1.0):
    """x [tokens][heads][dim], dims [0, 2 len(inv_freq)) turned."""
    pairs = len(inv_freq)
    x = np.asarray(x, np.float64)
    if pairs == 0:
        return x.copy()
    angle = np.asarray(positions, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    out = x.copy()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        out[..., :pairs], out[..., pairs:2 * pairs] = a * c - b * s, b * c + a * s
    return out


class Cache:
    """values: the numbers the codes stand for; keys / vals [page][head][token][dim]."""

    def __init__(self, heads, dim, page, capacity, fmt):
        self.heads, self.dim, self.page, self.capacity, self.fmt = heads, dim, page, capacity, fmt
        self.codes = [np.zeros((capacity, heads, page, dim)) for _ in range(2)]
        self.scales = [np.zeros((capacity, heads), np.float32) for _ in range(2)]
        self.summaries = np.zeros((capacity, heads * dim))
        self.counts = np.zeros(capacity, np.int32)

    def append(self, pages, past, keys, values):
        """keys, values [tokens][heads][dim], already rotated."""
        n, ps = len(keys), self.page
        with np.errstate(all="ignore"):
            self._append(pages, past, keys, values, n, ps)

    def _append(self, pages, past, keys, values, n, ps):
        for slot in range(past // ps, (past + n - 1) // ps + 1 if n else 0):
            page = pages[slot]
            o0, o1 = max(past - slot * ps, 0), min(past + n - slot * ps, ps)
            for side, x in enumerate((keys, values)):
                x = np.asarray(x, np.float64)[slot * ps + o0 - past:slot * ps + o1 - past].swapaxes(0, 1)
                most = np.abs(np.where(np.isfinite(x), x, 0)).max((1, 2))
                had = self.scales[side][page] if o0 else np.zeros(self.heads, np.float32)
                scale = np.maximum(had, scale_for(self.fmt, most))
                wide = scale.astype(np.float64)[:, None, None]
                mine = self.codes[side][page]
                grew = (scale > had)[:, None, None]
                brought = nearest(self.fmt, mine[:, :o0] * had.astype(np.float64)[:, None, None] / wide)
                mine[:, :o0] = np.where(grew, brought, mine[:, :o0])
                mine[:, o0:o1] = nearest(self.fmt, x / wide)
                self.scales[side][page] = scale
            mean = self.codes[0][page][:, :o1].mean(1) * self.scales[0][page].astype(np.float64)[:, None]
            self.summaries[page] = mean.reshape(-1)
            self.counts[page] = o1

    def rows(self, pages, tokens=None):
        """(keys, values) [heads][tokens][dim] of a list of pages: each page's
        count of tokens, or the first `tokens` of the list; and [heads][tokens],
        the largest number that a token's value scale has a code for."""
        if len(pages) == 0:
            empty = np.zeros((self.heads, 0, self.dim))
            return empty, empty, empty[..., 0]
        got = []
        most = np.repeat(self.scales[1][pages].astype(np.float64).T * LARGEST[self.fmt], self.page, 1)
        for side in range(2):
            x = self.codes[side][pages] * self.scales[side][pages].astype(np.float64)[:, :, None, None]
            x = x.swapaxes(0, 1).reshape(self.heads, -1, self.dim)
            if tokens is None:
                keep = (np.arange(self.page) < self.counts[pages][:, None]).reshape(-1)
                got.append(x[:, keep])
            else:
                got.append(x[:, :tokens])
        return got[0], got[1], most[:, keep] if tokens is None else most[:, :tokens]


def attend(q, keys, values, scale, sees=None, most=None):
    """softmax(scale q K^T) V of rows q [rows][dim] of one key head; row i sees
    the first sees[i] tokens.  Returns (out, sum p |v|, max |scale| sum |q k|,
    max p * most), most as Cache.rows gives it."""
    rows, tokens = len(q), keys.shape[0]
    if tokens == 0:
        zero = np.zeros((rows, values.shape[1]))
        return zero, zero, np.zeros(rows), np.zeros(rows)
    with np.errstate(all="ignore"):
        s = scale * (q @ keys.T)
        size = np.nan_to_num(np.abs(scale) * (np.abs(q) @ np.abs(keys).T)).max(1)
        if sees is not None:
            s = np.where(np.arange(tokens) < np.asarray(sees)[:, None], s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p = p / p.sum(1, keepdims=True)
        if sees is not None:
            p = np.where(np.arange(tokens) < np.asarray(sees)[:, None], p, 0.0)
        peak = np.zeros(rows) if most is None else (p * most).max(1)
        return p @ values, p @ np.abs(values), size, peak


def allowed(out, weighted, size, peak, dim, tokens, kind):
    """How far an output may be from the 64-bit one, element by element.

    A logit is a dot of exact products (8-bit codes times 11-bit halves of q)
    summed in float32 over dim terms and scaled three times, the query being held
    to 2^-21 of each element where it is float32 (two halves): its error is at
    most (dim + 8) 2^-24 + 2^-21 of sum |q k|.  Exponentials take twice that as a
    relative error (the row's maximum moves too) and 2^-21 of their own; a weight
    is rounded to 2^-11 (one half) or 2^-21 (two); sums over the tokens add
    tokens * 2^-24, numerator and denominator each.  All of it acts on sum p |v|.
    A weight (times its page's scale) is held so that the row's largest lies in
    [2^11, 2^15], and a half's numbers end in steps of 2^-24: each token's is off
    by half a step, 2^-25 / 2^11 = 2^-36 of the largest, besides, times a code of
    at most peak over it.
    The output is rounded once, by half a step of its type.  2^-126: results
    below the normal numbers."""
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[kind]
    logit = ((dim + 8) * 2.0 ** -24 + 2.0 ** -21) * size
    weight = 2.0 ** -11 if kind == "bf16" else 2.0 ** -21
    rel = 4 * logit + 2 * (2.0 ** -21 + tokens * 2.0 ** -24) + weight
    floor = 2.0 ** -24 if kind == "f16" else 2.0 ** -126
    least = (tokens * 2.0 ** -36 * peak)[:, None] if tokens else 0.0
    return half * np.abs(out) + rel[:, None] * (1 + half) * weighted + least + floor
