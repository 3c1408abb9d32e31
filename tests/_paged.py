"""Paged caches for the tests: random pools and tables on a device, and the same as the oracle takes them."""

from __future__ import annotations

import numpy as np
import torch

from oracle import paged_ref

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def host(t: torch.Tensor) -> np.ndarray:
    return t.double().cpu().numpy()


def typed(dtype):
    return lambda a: host(torch.from_numpy(np.asarray(a, np.float64)).to(torch.float32).to(dtype))


def make_pages(g, pool, Hk, P, D, dtype, bits, dev, spread=1.0):
    """Keys or values of a pool: bf16 / fp16 normal values, or codes with a scale for each page and head."""
    x = torch.randn(pool, Hk, P, D, generator=g) * spread
    if bits == 16:
        return x.to(dtype).to(dev)
    codes = (x * 90 / spread).clamp_(-448, 448).to(torch.float8_e4m3fn)
    e = torch.randint(-9, -4, (pool, Hk), generator=g)
    return codes.to(dev), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(dev)


def exps(scales: torch.Tensor) -> np.ndarray:
    return scales.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64) - 127


def oracle_pages(pages) -> paged_ref.Pages:
    if isinstance(pages, tuple):
        e = exps(pages[1])
        return paged_ref.Pages(host(pages[0]) * np.exp2(e.astype(np.float64))[:, :, None, None], e)
    return paged_ref.Pages(host(pages))


def make_table(g, lens, P, pool, dev, more=2):
    """Random distinct pages for sequences of these lengths; -1 behind them."""
    used = [max(0, -(-n // P)) for n in lens]
    assert sum(used) <= pool
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(used + [0]) + more), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    return table.to(dev)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def starts_of(rows, dev):
    return ints([0] + np.cumsum(rows).tolist(), dev)


def attention(q, k, v, table, starts, lens, scale, causal=True, pieces=2.0 ** -16):
    """The oracle's attention for many keys (float64, rows of no sequence NaN), and how far a kernel's may be off before its last
    rounding. Scores are sums of D exact products in fp32, each sum off by 2^-24 of the sizes so far: D 2^-24 sum |q k| together,
    times the scale (and 2^-22 of the exponent itself, which is a product and a power of two) in a probability, numerator and
    denominator; the probabilities' pieces are off by ``pieces`` of their values, and sums over keys in fp32 by 2^-24 a step of
    32 keys and of every join: 2^-24 (keys / 32 + 64)."""
    T, Hq, D = q.shape
    pool, Hk, P, _ = k.values.shape
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b, s0, n, p0 in paged_ref.sequences(table, starts, lens, T):
        p = np.arange(min(int(lens[b]), table.shape[1] * P))
        ids = table[b][p // P]
        there = (ids >= 0) & (ids < pool)
        p, ids = p[there], ids[there]
        seen = (p[None] <= p0 + np.arange(n)[:, None]) if causal else np.ones((n, p.size), bool)
        for h in range(Hq):
            g = h // (Hq // Hk)
            kk, vv, qq = k.values[ids, g, p % P], v.values[ids, g, p % P], q[s0:s0 + n, h]
            s = np.where(seen, qq @ kk.T * scale, -np.inf)
            top = s.max(-1, keepdims=True, initial=-1e300)
            w = np.exp(s - top)
            total = w.sum(-1, keepdims=True)
            w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
            out[s0:s0 + n, h] = w @ vv
            size = np.where(seen, np.abs(qq) @ np.abs(kk).T * scale, 0).max(-1, initial=0)
            far = np.where(seen & (w > 2.0 ** -40), top - s, 0).max(-1, initial=0)
            e = 2 * (D * 2.0 ** -24 * 2 * size + 2.0 ** -22 * (1 + far)) + pieces + 2.0 ** -24 * (p.size / 32 + 64)
            tol[s0:s0 + n, h] = e[:, None] * (w @ np.abs(vv))
    return out, tol


def check_rows(got, want, tol):
    """got: a tensor; one rounding to its type on top of ``tol``. Rows of no sequence (NaN in want) are zeros."""
    fi = torch.finfo(got.dtype)
    got, none = host(got), np.isnan(want)
    assert not got[none].any()
    w = np.where(none, 0.0, want)
    limit = tol + (np.abs(w) + tol) * fi.eps / 2 + fi.smallest_normal * fi.eps
    assert (np.abs(got - w) <= limit).all(), float((np.abs(got - w) / limit).max())
