"""Operators of serving many sequences from a paged cache, each in its plain form and as the framework's own call.

* ``append``: the rows of a step (decoded tokens, verify blocks, prompt chunks of several sequences, one after the
  other) rotated to their positions, queries handed on, keys and values written into their sequences' pages, in the
  model's type or in 8 bits (e4m3 codes with one power-of-two scale for each page and head);
* ``attend``: those queries over their sequences' pages, whatever mixture of row counts and lengths a step has;
* ``score``: log probabilities of given tokens, the entropy of their distributions and the best alternatives.

``own`` false: elementary torch operations. ``own`` true: the calls of ``dspark_rocm.ops``.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE = torch.float8_e4m3fn
SCALE = torch.float8_e8m0fnu
LEAST = -110            # the smallest exponent of a page's scale


def _ops():
    try:
        from dspark_rocm import ops
    except ImportError:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-dspark_amd"))
        from dspark_rocm import ops
    return ops


# ------------------------------------------------------------------ the cases


def listed():
    # a sequence has between `short` and `long` tokens in the cache, this step's among them, and between `few` and
    # `many` rows in this step
    return [
        # the next token of one user
        dict(name="append_one", kind="append", batch=1, few=1, many=1, short=1000, long=1000, hq=32, hk=8, d=128, page=64,
             bits=16, dtype="bf16", dims=128, interleaved=False, base=1e6),
        # a decode step of a serving batch into 8-bit pages
        dict(name="append_step8", kind="append", batch=48, few=1, many=1, short=20, long=2000, hq=32, hk=8, d=128, page=16,
             bits=8, dtype="bf16", dims=128, interleaved=False, base=5e5),
        # a prompt chunk behind an earlier one
        dict(name="append_chunk", kind="append", batch=1, few=2048, many=2048, short=3001, long=3001, hq=64, hk=8, d=128,
             page=64, bits=16, dtype="bf16", dims=128, interleaved=False, base=1e6),
        # prompts of three users into 8-bit pages: wide heads, half of each rotated, pairs side by side
        dict(name="append_chunk8", kind="append", batch=3, few=77, many=600, short=601, long=1999, hq=24, hk=4, d=256, page=64,
             bits=8, dtype="f16", dims=128, interleaved=True, base=1e4),
        # the next token of one user, just after a short prompt: latency is all it costs
        dict(name="attend_one", kind="attend", batch=1, few=1, many=1, short=129, long=129, hq=32, hk=8, d=128, page=16, bits=16,
             dtype="bf16"),
        # a decode step of a serving batch of unequal lengths
        dict(name="attend_decode", kind="attend", batch=32, few=1, many=1, short=90, long=8192, hq=32, hk=8, d=128, page=64,
             bits=16, dtype="bf16"),
        # two users at a long context, 8-bit pages
        dict(name="attend_long8", kind="attend", batch=2, few=1, many=1, short=70001, long=100000, hq=64, hk=8, d=128, page=128,
             bits=8, dtype="bf16"),
        # verify blocks of several users: up to 16 rows each, wide heads
        dict(name="attend_verify", kind="attend", batch=6, few=3, many=16, short=1500, long=10007, hq=24, hk=4, d=256, page=32,
             bits=16, dtype="f16"),
        # a long prompt's second chunk
        dict(name="attend_chunk", kind="attend", batch=1, few=2048, many=2048, short=5001, long=5001, hq=32, hk=8, d=128, page=64,
             bits=16, dtype="bf16"),
        # a prompt chunk scheduled together with users that decode, 8-bit pages
        dict(name="attend_mixed8", kind="attend", batch=7, few=1, many=700, short=700, long=6000, hq=16, hk=4, d=128, page=64,
             bits=8, dtype="bf16"),
        # what a sampled token is reported with: one row
        dict(name="score_one", kind="score", rows=1, vocab=151936, top=20, dtype="bf16", temperature=1.0),
        # a prompt scored token by token, an odd vocabulary (rows start unaligned)
        dict(name="score_prompt", kind="score", rows=900, vocab=128255, top=5, dtype="bf16", temperature=1.0),
    ]


def _log(rng, lo, hi):
    return min(max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))), hi)


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "score"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "score":
        vocab = _log(rng, 1000, 200000)
        return dict(kind=kind, rows=min(_log(rng, 1, 4096), 110000000 // vocab), vocab=vocab, top=rng.choice([0, rng.randint(1, 20), 64]),
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), temperature=rng.choice([1.0, 1.0, 0.7]))
    hq, hk, d = rng.choice([(32, 8, 128), (64, 8, 128), (24, 4, 256), (16, 8, 256), (8, 2, 64), (16, 4, 128), (9, 3, 64)])
    case = dict(kind=kind, hq=hq, hk=hk, d=d, page=rng.choice([16, 32, 64, 128]), bits=rng.choice([8, 16]), dtype=dtype)
    shape = rng.choice(["decode", "verify", "chunk", "mixed"])
    # no more rows together, nor longer sequences, than what the largest listed cases multiply, move and read
    total = 16000000 // ((hq + 2 * hk) * d) if kind == "append" else 6400000 // (hq * d)
    if shape == "decode":
        batch, few, many = _log(rng, 1, 64), 1, 1
    elif shape == "verify":
        batch, few, many = _log(rng, 1, 16), rng.randint(1, 4), rng.randint(4, 16)
    elif shape == "chunk":
        batch = rng.randint(1, 2)
        few = many = _log(rng, 17, total // batch)
    else:
        batch, few, many = rng.randint(2, 6), 1, _log(rng, 17, min(600, total // 4))
    most = 60000 if kind == "append" else (100000 if shape == "decode" else 10000 if shape == "verify" else 5000)
    room = (24 << 20) if kind == "append" else (160 << 20)
    long = max(many, _log(rng, many + 1, max(many + 1, min(most, room // (batch * hk * d)))))
    short = max(many, _log(rng, many, long))
    case.update(batch=batch, few=few, many=many, short=short, long=long)
    if kind == "append":
        case.update(dims=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.4, base=rng.choice([1e4, 5e5, 1e6, 1e7]))
    return case


def _spread(lo, hi, n, turn):
    """n whole numbers from lo to hi in no order, the last one hi: fixed by the case."""
    return [lo + int((hi - lo) * ((i * turn + turn) % 1.0)) for i in range(n - 1)] + [hi]


def _rows(case):
    return _spread(case["few"], case["many"], case["batch"], 0.6180339887)


def _lens(case):
    return _spread(case["short"], case["long"], case["batch"], 0.7548776662)


# ------------------------------------------------------------------ inputs


def _pages(g, case, n, kind):
    """n pages [n, Hk, page, D] of keys or values: of the model's type, or e4m3 codes and the pages' scales."""
    shape = (n, case["hk"], case["page"], case["d"])
    if case["bits"] == 16:
        return torch.randn(shape, generator=g, device=DEV, dtype=DTYPES[case["dtype"]]) * (1.0 if kind == "k" else 0.5)
    codes = (torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16) * 96).clamp_(-448, 448).to(CODE)
    up = torch.randint(-8, -5, shape[:2], generator=g, device=DEV)
    return codes, (up + 127).to(torch.uint8).view(SCALE)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "score":
        n, V = case["rows"], case["vocab"]
        # most of the vocabulary near the mean, a few tokens that stand out, some that a grammar forbids
        x = torch.randn((n, V), generator=g, device=DEV) * 2.0
        top = torch.randint(0, V, (n, 24), generator=g, device=DEV)
        x.scatter_add_(1, top, 4.0 + 5.0 * torch.rand((n, 24), generator=g, device=DEV))
        x.masked_fill_(torch.rand((1, V), generator=g, device=DEV) < 0.01, -math.inf)
        st["tokens"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.8, x.argmax(-1), top[:, 0])
        st["logits"] = x.to(DTYPES[case["dtype"]])
        return st
    rows, lens, page, d = _rows(case), _lens(case), case["page"], case["d"]
    dt, T, B = DTYPES[case["dtype"]], sum(_rows(case)), case["batch"]
    used = [-(-n // page) for n in lens]
    pool = sum(used) + 3
    ids = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(used) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    st["table"] = table
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["starts"] = torch.tensor([0] + np.cumsum(rows).tolist(), dtype=torch.int32, device=DEV)
    st["longest"], st["most"] = max(lens), max(rows)
    st["k_pages"], st["v_pages"] = _pages(g, case, pool, "k"), _pages(g, case, pool, "v")
    if case["kind"] == "attend":
        st["q"] = torch.randn((T, case["hq"], d), generator=g, device=DEV).mul_(1.3).to(dt)
        return st
    # one projection's output, as a layer makes it; its heads are views
    x = torch.randn((T, (case["hq"] + 2 * case["hk"]) * d), generator=g, device=DEV)
    x *= torch.exp(0.4 * torch.randn((T, 1), generator=g, device=DEV))
    st["q"], st["k"], st["v"] = (t.unflatten(1, (-1, d)) for t in x.to(dt).split([case["hq"] * d, case["hk"] * d, case["hk"] * d], 1))
    i = torch.arange(case["dims"] // 2, dtype=torch.float64, device=DEV)
    st["freqs"] = torch.exp2(i * (-2.0 / case["dims"] * math.log2(case["base"])))
    if case["bits"] == 8:
        # the pages this step writes into: what a program looks at that keeps its pages elsewhere too
        st["touched"] = torch.cat([table[b, (n - r) // page:(n - 1) // page + 1] for b, (n, r) in enumerate(zip(lens, rows))])
    return st


# ------------------------------------------------------------------ one pass


def _where(st):
    """Of every row: its sequence and its position in it."""
    starts, lens = st["starts"].long(), st["lens"].long()
    t = torch.arange(st["q"].shape[0], device=DEV)
    b = torch.searchsorted(starts[1:], t, right=True)
    return b, lens[b] - starts[b + 1] + t


def _rotated(x, pos, freqs, interleaved):
    """Angles in 64 bits, their sines and cosines rounded to 32, then three operations in 32 bits."""
    half = freqs.numel()
    ang = pos.double()[:, None, None] * freqs
    c, s = torch.cos(ang).float(), torch.sin(ang).float()
    r, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * c - b * s, a * s + b * c
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y.to(x.dtype), rest], -1)


def _up(scales):
    return scales.view(torch.uint8).int() - 127


def _write8(pages, x, page, off, touched):
    """Rows x [T, Hk, D] into 8-bit pages: a page's exponent is the least that fits its new rows and no less than that of the
    rows that it held before them, which are rescaled where it grew."""
    codes, scales = pages
    P, H = scales.shape
    xf = x.float()
    amax = torch.zeros((P, H), device=DEV).index_reduce_(0, page, xf.abs().amax(-1), "amax")
    first = torch.full((P,), codes.shape[2], device=DEV).index_reduce_(0, page, off, "amin")
    m, e = torch.frexp(amax)                                    # amax = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    need = torch.where(amax > 0, e - 9 + (m > 0.875).int(), LEAST).clamp(min=LEAST)
    old = torch.where((first > 0)[:, None], _up(scales), LEAST)
    new = torch.maximum(need, old)[touched]
    shift = torch.exp2((old[touched] - new).float())[..., None, None]
    kept = codes[touched].float()
    held = torch.arange(codes.shape[2], device=DEV) < first[touched, None]
    codes[touched] = torch.where(held[:, None, :, None], kept * shift, kept).to(CODE)
    scales.view(torch.uint8)[touched] = (new + 127).to(torch.uint8)
    codes[page, :, off] = (xf * torch.exp2(-_up(scales)[page].float())[..., None]).to(CODE)


def _values(pages, at, dtype):
    """Pages `at` as the values that they stand for."""
    if isinstance(pages, tuple):
        codes, scales = pages
        return (codes[at].float() * torch.exp2(_up(scales)[at].float())[..., None, None]).to(dtype)
    return pages[at].to(dtype)


def _plain_append(st, case):
    b, pos = _where(st)
    P = case["page"]
    page, off = st["table"][b, pos // P].long(), pos % P
    q, k = (_rotated(st[n], pos, st["freqs"], case["interleaved"]) for n in ("q", "k"))
    if case["bits"] == 16:
        st["k_pages"][page, :, off] = k
        st["v_pages"][page, :, off] = st["v"]
        return q, st["k_pages"], st["v_pages"]
    touched = st["touched"].long()
    _write8(st["k_pages"], k, page, off, touched)
    _write8(st["v_pages"], st["v"], page, off, touched)
    return q, _values(st["k_pages"], touched, q.dtype), _values(st["v_pages"], touched, q.dtype)


def _plain_attend(st, case):
    B, P, H, d = case["batch"], case["page"], case["hk"], case["d"]
    L, n, g = st["longest"], st["most"], case["hq"] // case["hk"]
    at = st["table"][:, :-(-L // P)].long().clamp(min=0)
    k, v = (_values(st[t], at, torch.float32).transpose(1, 2).flatten(2, 3)[:, :, :L] for t in ("k_pages", "v_pages"))
    starts, lens = st["starts"].long(), st["lens"].long()
    i = torch.arange(n, device=DEV)
    row = (starts[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][row].float().unflatten(2, (H, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [B, H, g * n, d]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * d ** -0.5
    last = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + i                              # of row i, [B, n]
    seen = torch.arange(L, device=DEV) <= last[..., None]
    s = s.unflatten(2, (g, n)).masked_fill(~seen[:, None, None], -math.inf).flatten(2, 3)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.unflatten(2, (g, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)                             # [B, n, H * g, d]
    b, _ = _where(st)
    return o[b, torch.arange(st["q"].shape[0], device=DEV) - starts[b]].to(st["q"].dtype)


def _plain_score(st, case):
    x = st["logits"].float() / case["temperature"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * (x - top), 0.0).sum(-1) / total
    given = (x.gather(-1, st["tokens"][:, None]) - top)[:, 0] - log_total
    if not case["top"]:
        none = given.new_zeros((x.shape[0], 0))
        return given, entropy, none.int(), none
    order = torch.sort(st["logits"], dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    return given, entropy, order.int(), (x.gather(-1, order) - top) - log_total[:, None]


def run(st):
    case = st["case"]
    if case["kind"] == "score":
        if own:
            return _ops().token_logprobs(st["logits"], st["tokens"], top=case["top"], temperature=case["temperature"])
        return _plain_score(st, case)
    if case["kind"] == "attend":
        if own:
            return _ops().paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["starts"], st["lens"],
                                          scale=case["d"] ** -0.5, max_rows=st["most"], max_len=st["longest"])
        return _plain_attend(st, case)
    if own:
        ops = _ops()
        q = ops.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["starts"], st["lens"],
                             q=st["q"], freqs=st["freqs"], interleaved=case["interleaved"])
        if case["bits"] == 16:
            return q, st["k_pages"], st["v_pages"]
        return (q, *ops.paged_read(st["k_pages"], st["v_pages"], st["touched"], dtype=q.dtype))
    return _plain_append(st, case)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["kind"] == "score":
        n = case["rows"] * case["vocab"]
        # the logits once; an exponential (8 operations), two sums, a comparison for each
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (16 + 8 * case["top"]), "flops": 12 * n}
    rows, lens, page = _rows(case), _lens(case), case["page"]
    T, per, kept = sum(rows), 2 * case["hk"] * case["d"], case["bits"] // 8
    ids = 4 * (sum(-(-n // page) for n in lens) + 2 * case["batch"] + 1)
    if case["kind"] == "append":
        # queries read and written, keys and values read and written; 8-bit pages: the touched ones read back
        b = T * (2 * 2 * case["hq"] * case["d"] + per * (2 + kept))
        if case["bits"] == 8:
            b += sum((n - 1) // page - (n - r) // page + 1 for n, r in zip(lens, rows)) * page * per * (kept + 2)
        return {"bytes": b, "flops": 3 * T * (case["hq"] + case["hk"]) * case["dims"] + 20 * T * case["dims"]}
    seen = sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, rows))
    return {"bytes": 2 * 2 * T * case["hq"] * case["d"] + sum(lens) * per * kept + ids,
            "flops": 4 * case["hq"] * case["d"] * seen}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits


def _e4m3(x):
    """numpy float64 of at most 448 in size -> the nearest e4m3 value, halves to the even one."""
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -40))), -6.0)
    step = np.exp2(e - 3.0)
    return np.round(x / step) * step


def _host(t):
    return t.double().cpu().numpy()


def _exact_append(st, case):
    P, half = case["page"], case["dims"] // 2
    rows, lens, table = _rows(case), _lens(case), st["table"].cpu().numpy()
    f32, typed = (lambda a: a.astype(np.float32)), (lambda a: _host(torch.from_numpy(a).to(DTYPES[case["dtype"]])))
    first = np.arange(half) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
    ang = pos.astype(np.float64)[:, None, None] * st["freqs"].cpu().numpy()
    c, s = f32(np.cos(ang)), f32(np.sin(ang))                   # the definition's steps from here on are in 32 bits
    outs = {}
    for name in ("q", "k"):
        x = _host(st[name])
        a, b, y = f32(x[..., first]), f32(x[..., second]), x.copy()
        y[..., first], y[..., second] = a * c - b * s, a * s + b * c
        outs[name] = typed(y)
    outs["v"] = _host(st["v"])
    if case["bits"] == 16:
        ends = []
        for name in ("k", "v"):
            to = _host(st[name + "_pages"])
            t = 0
            for b, (n, r) in enumerate(zip(lens, rows)):
                for p in range(n - r, n):
                    to[table[b, p // P], :, p % P] = outs[name][t]
                    t += 1
            ends.append(to)
        return outs["q"], *ends
    ends = []
    for name in ("k", "v"):
        codes, scales = st[name + "_pages"]
        t, done = 0, []
        for b, (n, r) in enumerate(zip(lens, rows)):
            at = n - r
            while at < n:
                p, lo = table[b, at // P], at % P
                hi = min(P, lo + n - at)
                x = outs[name][t:t + hi - lo].transpose(1, 0, 2)                        # [Hk, new rows, D]
                e = np.ceil(np.log2(np.maximum(np.abs(x).max((1, 2)), 1e-300) / 448.0))
                e = np.maximum(e, LEAST)
                was = scales[p].view(torch.uint8).cpu().numpy().astype(np.float64) - 127
                if lo:
                    e = np.maximum(e, was)
                unit, old = np.exp2(e)[:, None, None], np.exp2(was)[:, None, None]
                v = _host(codes[p])
                v[:, :lo] = _e4m3(v[:, :lo] * (old / unit))
                v[:, lo:hi] = _e4m3(x / unit)
                done.append(v * unit)
                t, at = t + hi - lo, at + hi - lo
        ends.append(np.stack(done))
    return outs["q"], *ends


def _exact_attend(st, case):
    P, g, d = case["page"], case["hq"] // case["hk"], case["d"]
    out, t = torch.zeros(st["q"].shape, dtype=torch.float64), 0

    def head(pages, ids, h, n):
        if isinstance(pages, tuple):
            x = pages[0][ids, h].double() * torch.pow(2.0, pages[1].view(torch.uint8)[ids, h].double() - 127.0)[:, None, None]
        else:
            x = pages[ids, h].double()
        return x.reshape(-1, d)[:n]

    for b, (n, r) in enumerate(zip(_lens(case), _rows(case))):
        ids = st["table"][b, :-(-n // P)].long()
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - r, n, device=DEV)[:, None]
        for h in range(case["hq"]):
            k, v = head(st["k_pages"], ids, h // g, n), head(st["v_pages"], ids, h // g, n)
            s = st["q"][t:t + r, h].double() @ k.t().contiguous() / math.sqrt(d)
            out[t:t + r, h] = (torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v).cpu()
        t += r
    return out.numpy()


def _exact_score(st, case):
    n, top = case["rows"], case["top"]
    given, entropy = np.zeros(n), np.zeros(n)
    ids, best = np.zeros((n, top), np.int32), np.zeros((n, top))
    tokens = st["tokens"].cpu().numpy()
    for i in range(n):
        x = _host(st["logits"][i]) / case["temperature"]
        z = x - x.max()
        lse = math.log(np.exp(z).sum())
        lp = z - lse
        p = np.exp(lp)
        given[i] = lp[tokens[i]]
        entropy[i] = -(p[p > 0] * lp[p > 0]).sum()
        if top:
            least = np.partition(x, -top)[-top]
            some = np.nonzero(x >= least)[0]
            some = some[np.argsort(-x[some], kind="stable")][:top]
            ids[i], best[i] = some, lp[some]
    return given, entropy, ids, best


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "score": _exact_score}[case["kind"]](st, case)
