"""The quantised paged K/V cache in plain numpy, 64 bits: what its rows stand
for after any appends, and attention over them.  A block is one page of one
head; its values are payload * 2^(code - 127)."""
from __future__ import annotations

import numpy as np
import torch

LARGEST = {"int8": 127.0, "e4m3": 448.0}
TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def code_of(amax, fmt):
    """Scale byte of a block of this largest magnitude."""
    if not amax <= LARGEST[fmt] * 2.0 ** (121 if fmt == "int8" else 119):
        return 255  # no finite number, or one whose payload could stand for 2^128
    e = -126
    while amax > LARGEST[fmt] * 2.0 ** e:
        e += 1
    return e + 127


def round_payload(y, fmt):
    """Nearest payload, ties to even (y within the payload's range)."""
    if fmt == "int8":
        return np.rint(y)
    _, ex = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(ex, -5) - 4)
    return np.rint(y / step) * step


class Cache:
    """payload [pages, heads, rows, dim] and code [pages, heads], as numbers."""

    def __init__(self, pages, heads, rows, dim, fmt, payload=None, code=None):
        self.fmt, self.rows = fmt, rows
        self.payload = np.zeros((pages, heads, rows, dim)) if payload is None else payload
        self.code = np.zeros((pages, heads), np.int64) if code is None else code

    @staticmethod
    def of(cache):
        """The contents of an ops.QuantPagedCache."""
        fmt = "int8" if cache.pool.dtype == torch.int8 else "e4m3"
        pages, heads, rows, dim = cache.pool.shape
        return Cache(pages, heads, rows, dim, fmt, cache.pool.cpu().float().double().numpy(),
                     cache.scales.cpu().numpy().astype(np.int64))

    def append(self, x, table, pos, counts):
        """x [B, heads, T, dim]."""
        for b in range(x.shape[0]):
            done = 0
            while done < counts[b]:
                page, r0 = divmod(int(pos[b]) + done, self.rows)
                n = min(self.rows - r0, counts[b] - done)
                block = table[b][page]
                for h in range(x.shape[1]):
                    new = np.asarray(x[b, h, done:done + n], np.float64)
                    was = int(self.code[block, h]) if r0 else 0
                    code = max(code_of(np.abs(new).max() if np.isfinite(new).all() else np.inf, self.fmt), was)
                    kept = self.payload[block, h, :r0]
                    if r0 and code > was and code != 255:
                        kept[:] = round_payload(np.ldexp(kept, was - code), self.fmt)
                    self.payload[block, h, r0:r0 + n] = (
                        0.0 if code == 255 else round_payload(np.ldexp(new, 127 - code), self.fmt))
                    self.code[block, h] = code
                done += n

    def rows_of(self, table_row, first, n):
        """Values of rows first .. first + n [heads, n, dim]."""
        at = np.arange(first, first + n)
        blocks = np.asarray(table_row)[at // self.rows]
        scale = np.where(self.code == 255, np.nan, np.ldexp(1.0, np.where(self.code == 255, 0, self.code) - 127))
        v = self.payload[blocks, :, at % self.rows] * scale[blocks][..., None]
        return v.transpose(1, 0, 2)


def attention(q, k, v, table, pos, counts, window, scale, weight=0.0):
    """(out, slack) [B, Hq, T, D]: slack bounds the error of fp32 arithmetic.

    With u = 2^-24: a score of D products has error at most (D + 4) u sum|q||k|
    scale, the exponent's own rounding (the score times log2 e, less the
    maximum, two roundings and exp2) 4 u (|s| + |m| + 1); p is off by those
    relatively, in the weights and in their sum; a weighted sum of n terms adds
    (n + 16) u of sum p|v|, and weights held to a relative `weight` that much more.
    Weights are at most 1 and fp32's normal numbers end at 2^-126: one below that
    may be 0, so each of n terms is also off by up to 2^-126 max|v|, over a sum of
    weights of at least 1."""
    B, hq, T, D = q.shape
    heads = k.payload.shape[1]
    scale = 1.0 / np.sqrt(D) if scale <= 0 else scale
    u = 2.0 ** -24
    out, slack = np.zeros(q.shape), np.zeros(q.shape)
    cap = len(table[0]) * k.rows
    for b in range(B):
        n = min(int(pos[b]) + int(counts[b]), cap)
        if n <= 0 or counts[b] <= 0:
            continue
        lo = max(0, int(pos[b]) - window + 1) if window else 0
        kk, vv = k.rows_of(table[b], lo, n - lo), v.rows_of(table[b], lo, n - lo)
        at = np.arange(lo, n)
        for t in range(int(counts[b])):
            last = int(pos[b]) + t
            see = (at <= last) & ((at > last - window) if window else True)
            if not see.any():
                continue
            for h in range(hq):
                kh, vh = kk[h // (hq // heads)][see], vv[h // (hq // heads)][see]
                s = kh @ q[b, h, t] * scale
                m = s.max()
                p = np.exp(s - m)
                out[b, h, t] = p @ vh / p.sum()
                ds = (D + 4) * u * (np.abs(kh) @ np.abs(q[b, h, t])).max() * abs(scale)
                rel = 2 * (ds + 4 * u * (2 * np.abs(s).max() + 1)) + (len(s) + 16) * u + weight
                slack[b, h, t] = rel * (p @ np.abs(vh)) / p.sum() + len(s) * 2.0 ** -126 * np.abs(vh).max()
    return out, slack


def assert_attention(got, want, slack, what=""):
    """got within its type's rounding (half a step of the value) of want, give or take slack."""
    g = got.detach().cpu().double().numpy()
    half = torch.finfo(got.dtype).eps / 2
    assert g.shape == want.shape
    np.testing.assert_array_equal(np.isnan(g), np.isnan(want), err_msg=f"{what}: NaN")
    err = np.abs(g - want)
    bound = half * (np.abs(want) + slack) + slack + 1e-37
    bad = np.isfinite(want) & ~(err <= bound)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, err / bound, 0)), err.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; worst at {i}: got {g[i]!r} want {want[i]!r} "
                             f"bound {bound[i]:.3g}")
