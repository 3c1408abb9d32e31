"""Sampling from next-token logits in 64 bits: the truncated softmax and the accept rule of a sampled
speculative round (the reference's ``truncate_probs``, sampling.py, and its sampling accept, generate.py).
Plain loops over rows and tokens; test infrastructure only.
"""

from __future__ import annotations

import numpy as np


def weights(x, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0) -> np.ndarray:
    """float64 weights of one row ``x`` [V], 0 for every token that is cut."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.exp((x - top) / temperature)
    if (top_k == 0 or top_k >= x.size) and top_p >= 1.0:
        return w
    order = np.argsort(-x, kind="stable")               # equal logits (0 and -0 too) by index
    if top_k:
        order = order[:top_k]
    if top_p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[before[:-1] < top_p * before[-1]]
    out = np.zeros_like(w)
    out[order] = w[order]
    return out


def probs(x, **kw) -> np.ndarray:
    w = weights(x, **kw)
    s = w.sum()
    return w / s if s > 0 else w


def verify(logits, draft, uniforms, draft_probs=None, lens=None, **kw):
    """logits [B, m + 1, V] -> (n [B], tokens [B, m + 1], draft_p [B, m])."""
    B, R, V = logits.shape
    m = R - 1
    n, tokens, px = np.zeros(B, np.int32), np.full((B, R), -1, np.int32), np.zeros((B, m))
    for b in range(B):
        ps = [probs(logits[b, i], **kw) for i in range(R)]
        for i in range(m):
            if 0 <= draft[b, i] < V:
                px[b, i] = ps[i][draft[b, i]]
        length = m if lens is None else min(max(int(lens[b]), 0), m)
        k = 0
        while k < length:
            d = int(draft[b, k])
            q = 1.0 if draft_probs is None else float(draft_probs[b, k, d]) if 0 <= d < V else 0.0
            if not float(uniforms[b, k]) * q < px[b, k]:
                break
            k += 1
        r = ps[k].copy()
        if k < length:
            q = np.zeros(V)
            if draft_probs is not None:
                q = np.asarray(draft_probs[b, k], np.float64)
            elif 0 <= draft[b, k] < V:
                q[draft[b, k]] = 1.0
            rest = np.maximum(r - q, 0.0)
            r = rest if rest.sum() > 0 else r
        cum = np.cumsum(r)
        over = np.nonzero(cum > float(uniforms[b, m]) * cum[-1])[0]
        token = int(over[0]) if over.size else int(np.nonzero(r)[0][-1]) if r.any() else 0
        n[b] = k
        tokens[b, :k] = draft[b, :k]
        tokens[b, k] = token
    return n, tokens, px
