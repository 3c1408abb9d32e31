"""Paged caches of many sequences in plain loops: rows appended (rotated, in the model's type or as 8-bit codes), attention
over a sequence's pages, and the log probabilities of tokens. 64 bits but where a rule names its roundings; test
infrastructure only.
"""

from __future__ import annotations

import numpy as np

LEAST = -110


def e4m3(x) -> np.ndarray:
    """The nearest e4m3 value (4 significant bits, unit 2^-9, up to 448) of float64 ``x``, halves to even; NaN for what
    has none: NaN, and sizes that round past 448."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -60))), -6.0) - 3.0)
        y = np.round(x / step) * step
    return np.where(np.abs(y) <= 448.0, y, np.nan)


def rotate(x, pos, freqs, interleaved=False, scale=1.0, typed=lambda a: a) -> np.ndarray:
    """x [T, H, D] float64 (values of the model's type) at pos [T]; ``typed`` rounds float64 to that type."""
    half = len(freqs)
    ang = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = (np.cos(ang) * scale).astype(np.float32), (np.sin(ang) * scale).astype(np.float32)
    first = np.arange(half) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    a, b = x[..., first].astype(np.float32), x[..., second].astype(np.float32)
    y = np.array(x, np.float64)
    y[..., first] = typed((a * c - b * s).astype(np.float64))
    y[..., second] = typed((a * s + b * c).astype(np.float64))
    return y


def exponent(x, old: int | None) -> int:
    """The least E with |x| <= 448 2^E for the finite values of x, at least LEAST and ``old``."""
    x = np.abs(x[np.isfinite(x)])
    top = float(x.max()) if x.size else 0.0
    e = LEAST
    while top > 448.0 * 2.0 ** e:
        e += 1
    return e if old is None else max(e, old)


class Pages:
    """Keys or values: float64 values [pages, H, P, D], and for 8 bits exponents [pages, H]."""

    def __init__(self, values, exps=None):
        self.values, self.exps = np.array(values, np.float64), None if exps is None else np.array(exps, np.int64)

    def write(self, page: int, lo: int, rows) -> None:
        """rows [n, H, D] into page from its row ``lo`` on; rows before them are the sequence's, codes behind them stay."""
        n, H, _ = rows.shape
        if self.exps is None:
            self.values[page, :, lo:lo + n] = rows.transpose(1, 0, 2)
            return
        for h in range(H):
            e = exponent(rows[:, h], int(self.exps[page, h]) if lo else None)
            unit = 2.0 ** e
            with np.errstate(invalid="ignore"):
                self.values[page, h, :lo] = e4m3(self.values[page, h, :lo] / unit) * unit
                x = np.where(np.isfinite(rows[:, h]), rows[:, h], np.nan)
                self.values[page, h, lo:lo + n] = e4m3(x / unit) * unit
                self.values[page, h, lo + n:] *= unit / 2.0 ** int(self.exps[page, h])
            self.exps[page, h] = e


def sequences(table, starts, lens, T):
    """(b, first row, rows, first position, positions it can see) of every sequence with rows."""
    for b in range(len(lens)):
        s0, s1, n = int(starts[b]), int(starts[b + 1]), int(lens[b])
        if 0 <= s0 < s1 <= T and n > 0:
            yield b, s0, s1 - s0, n - (s1 - s0)


def append(pages: Pages, x, table, starts, lens) -> None:
    """x [T, H, D] (rotated) into the pages."""
    pool, _, P, _ = pages.values.shape
    for b, s0, n, p0 in sequences(table, starts, lens, x.shape[0]):
        i = 0
        while i < n:
            p = p0 + i
            if p < 0:
                i += 1
                continue
            m = min(n - i, P - p % P)
            if p // P < table.shape[1] and 0 <= table[b, p // P] < pool:
                pages.write(int(table[b, p // P]), p % P, x[s0 + i:s0 + i + m])
            i += m


def attention(q, k: Pages, v: Pages, table, starts, lens, scale, causal=True):
    """float64 [T, Hq, D], NaN in rows of no sequence; zeros where a row sees nothing."""
    T, Hq, D = q.shape
    pool, Hk, P, _ = k.values.shape
    out = np.full(q.shape, np.nan)
    for b, s0, n, p0 in sequences(table, starts, lens, T):
        keys = [(int(table[b, p // P]), p % P, p) for p in range(min(int(lens[b]), table.shape[1] * P))
                if 0 <= table[b, p // P] < pool]
        for i in range(n):
            seen = [(a, r) for a, r, p in keys if not causal or p <= p0 + i]
            out[s0 + i] = 0.0
            if not seen:
                continue
            a, r = (np.array(t) for t in zip(*seen))
            for h in range(Hq):
                g = h // (Hq // Hk)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k.values[a, g, r] @ q[s0 + i, h] * scale
                    w = np.exp(s - s.max())
                    out[s0 + i, h] = (w / w.sum()) @ v.values[a, g, r]
    return out


def logprobs(x, token: int, top: int = 0, temperature: float = 1.0):
    """One row of logits -> (log probability of ``token``, entropy, the ``top`` best tokens, theirs). NaN counts as -inf, an
    infinite logit takes all; tokens outside the row, and all of a row of nothing, have -inf."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    best = x.max()
    order = np.argsort(-x, kind="stable")[:top]
    if best == -np.inf:
        lp, entropy = np.full_like(x, -np.inf), 0.0
    else:
        with np.errstate(invalid="ignore"):
            z = np.where(x == best, 0.0, (x - best) / temperature) if best < np.inf else np.where(x == best, 0.0, -np.inf)
        lp = z - np.log(np.exp(z).sum())
        some = lp > -np.inf
        entropy = float(-(np.exp(lp[some]) * lp[some]).sum())
    return float(lp[token]) if 0 <= token < x.size else -np.inf, entropy, order, lp[order]
