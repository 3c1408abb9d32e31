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
