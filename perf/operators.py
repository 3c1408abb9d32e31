"""Operators of a sampled speculative round, each in its plain form and as the framework's own call.

* ``verify``: drafted tokens of a batch of sequences against the target's logits, from given random
  numbers: accepted counts, committed tokens, the target's probability of every drafted token;
* ``probs``: logits to the probabilities that are sampled from (temperature, top-k, top-p): what a
  drafter hands to ``verify`` beside its tokens;
* ``rope``: rotary positions of queries and keys, any pair layout, part of the head, positions of
  each row its own, as the rows of a draft tree have them;
* ``kv``: rows quantized into a cache as they are written, and the cache read back.

``own`` false: elementary torch operations. ``own`` true: the calls of ``dspark_rocm.ops``.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ops():
    try:
        from dspark_rocm import ops
    except ImportError:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-dspark_amd"))
        from dspark_rocm import ops
    return ops


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # the next token of one sequence: no draft, one row; launches are all it costs
        dict(name="sample_one", kind="verify", batch=1, draft=0, vocab=8192, dtype="bf16", temperature=0.8, top_k=40,
             top_p=1.0, q="none", ragged=False),
        # a verify step of one user: 15 drafts and the bonus row, the sampler most models ask for
        dict(name="verify_block", kind="verify", batch=1, draft=15, vocab=151936, dtype="bf16", temperature=0.6,
             top_k=20, top_p=0.95, q="dense", ragged=False),
        # drafts looked up in the prompt (no probabilities of their own), of unequal lengths, an odd vocabulary
        dict(name="verify_lookup", kind="verify", batch=5, draft=6, vocab=32003, dtype="f16", temperature=1.0, top_k=0,
             top_p=0.9, q="none", ragged=True),
        # a serving batch sampled from the whole distribution
        dict(name="verify_batch", kind="verify", batch=32, draft=7, vocab=151936, dtype="bf16", temperature=1.0,
             top_k=0, top_p=1.0, q="dense", ragged=False),
        # the drafter's own distributions for one block
        dict(name="probs_draft", kind="probs", rows=15, vocab=151936, dtype="bf16", temperature=0.7, top_k=0, top_p=0.9),
        # plain softmax at a temperature over a batch, an odd vocabulary (rows start unaligned)
        dict(name="probs_batch", kind="probs", rows=64, vocab=50257, dtype="f16", temperature=1.3, top_k=0, top_p=1.0),
        # one decoded token far into a long context
        dict(name="rope_decode", kind="rope", batch=1, rows=1, hq=32, hk=8, d=128, dims=128, interleaved=False,
             far=1000000, base=1e6, dtype="bf16", tree=False),
        # draft trees of a batch: positions by depth, a quarter of the head rotated
        dict(name="rope_tree", kind="rope", batch=6, rows=13, hq=24, hk=4, d=256, dims=64, interleaved=False,
             far=200000, base=1e7, dtype="f16", tree=True),
        # a prompt chunk with interleaved pairs
        dict(name="rope_prefill", kind="rope", batch=1, rows=2048, hq=64, hk=8, d=128, dims=128, interleaved=True,
             far=30000, base=1e4, dtype="bf16", tree=False),
        # a verify block appended to an 8-bit cache, which the stock attention then reads back
        dict(name="kv_verify", kind="kv", batch=1, heads=8, d=128, bits=8, rows=16, before=4001, dtype="bf16", out="f32"),
        # a prompt chunk into a 4-bit cache behind an earlier one
        dict(name="kv_chunk", kind="kv", batch=1, heads=4, d=256, bits=4, rows=2048, before=2953, dtype="bf16", out="bf16"),
        # one token at a long context
        dict(name="kv_long", kind="kv", batch=1, heads=8, d=128, bits=8, rows=1, before=32767, dtype="bf16", out="f32"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(max(step, int(round(v / step)) * step), hi)


def draw(rng):
    kind = rng.choice(["verify", "verify", "probs", "rope", "kv"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind in ("verify", "probs"):
        cut = rng.choice(["none", "k", "p", "both"])
        case = dict(kind=kind, vocab=_log(rng, 1000, 151936), dtype=dtype, temperature=round(rng.uniform(0.3, 1.5), 2),
                    top_k=_log(rng, 1, 200) if cut in ("k", "both") else 0,
                    top_p=round(rng.uniform(0.5, 0.99), 3) if cut in ("p", "both") else 1.0)
        most = 10 if cut != "none" else 20          # million logits: what is cut is sorted in the plain form
        if kind == "probs":
            return dict(case, rows=min(_log(rng, 1, 128), max(1, most * 1000000 // case["vocab"])))
        draft = rng.randint(0, 15)
        return dict(case, draft=draft, batch=min(_log(rng, 1, 32), max(1, most * 1000000 // (case["vocab"] * (draft + 1)))),
                    q=rng.choice(["none", "dense", "dense"]), ragged=rng.random() < 0.4)
    if kind == "rope":
        hq, hk, d = rng.choice([(32, 8, 128), (64, 8, 128), (24, 4, 256), (16, 8, 256), (8, 2, 64), (9, 3, 80)])
        tree = rng.random() < 0.4
        rows = rng.randint(1, 16) if tree else _log(rng, 1, 2048)
        return dict(kind=kind, batch=_log(rng, 1, 32) if rows <= 16 else 1, rows=rows, hq=hq, hk=hk, d=d,
                    dims=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.4, far=_log(rng, 100, 1000000),
                    base=rng.choice([1e4, 5e5, 1e6, 1e7]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), tree=tree)
    heads, d = rng.choice([(8, 128), (4, 256), (8, 256), (2, 64)])
    rows = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 2048)])
    batch = rng.choice([1, 1, 3])
    return dict(kind=kind, batch=batch, heads=heads, d=d, bits=rng.choice([4, 8]), rows=rows,
                before=_log(rng, 1, 30000 * 1024 // (batch * heads * d)), dtype=dtype, out=rng.choice(["f32", dtype]))


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(g, rows, case):
    """Next-token logits: most of the vocabulary near the mean, a few tokens that stand out."""
    x = torch.randn((rows, case["vocab"]), generator=g, device=DEV) * 2.0
    top = torch.randint(0, case["vocab"], (rows, 24), generator=g, device=DEV)
    return x.scatter_add_(1, top, 4.0 + 5.0 * torch.rand((rows, 24), generator=g, device=DEV))


def prepare(case, seed):
    g = _gen(seed)
    kind, st = case["kind"], {"case": case}
    if kind == "probs":
        st["logits"] = _logits(g, case["rows"], case).to(DTYPES[case["dtype"]])
    elif kind == "verify":
        B, m, V = case["batch"], case["draft"], case["vocab"]
        x = _logits(g, B * (m + 1), case).reshape(B, m + 1, V)
        st["logits"] = x.to(DTYPES[case["dtype"]])
        # the drafter's distribution: the target's with an error, cut by the same sampler; its token is drawn from it
        y = (x[:, :m] + 0.7 * torch.randn((B, m, V), generator=g, device=DEV)) / case["temperature"]
        if case["top_k"] and m:
            y = y.masked_fill(y < y.topk(min(case["top_k"], V), dim=-1).values[..., -1:], -math.inf)
        race = y - torch.log(-torch.log(torch.rand((B, m, V), generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)))
        st["draft"] = race.argmax(-1).to(torch.int32) if m else torch.zeros((B, 0), dtype=torch.int32, device=DEV)
        st["q"] = torch.softmax(y, -1) if case["q"] == "dense" and m else None
        st["uniforms"] = torch.rand((B, m + 1), generator=g, device=DEV)
        st["lens"] = torch.randint(0, m + 1, (B,), generator=g, device=DEV).to(torch.int32) if case["ragged"] else None
    elif kind == "rope":
        B, L, d = case["batch"], case["rows"], case["d"]
        dt = DTYPES[case["dtype"]]
        # projections as a layer makes them: [B, L, heads * d], seen as [B, heads, L, d]
        st["x"] = [torch.randn((B, L, h * d), generator=g, device=DEV).to(dt).view(B, L, h, d).transpose(1, 2)
                   for h in (case["hq"], case["hk"])]
        start = torch.randint(0, case["far"], (B, 1), generator=g, device=DEV)
        step = torch.randint(0, 7, (B, L), generator=g, device=DEV) if case["tree"] else torch.arange(L, device=DEV)[None]
        st["positions"] = start + step
        i = torch.arange(case["dims"] // 2, dtype=torch.float64, device=DEV)
        st["freqs"] = torch.exp2(i * (-2.0 / case["dims"] * math.log2(case["base"])))
    else:
        B, H, d, bits, n0, T = (case[k] for k in ("batch", "heads", "d", "bits", "before", "rows"))
        dt = DTYPES[case["dtype"]]
        cap = -(-(n0 + T) // 256) * 256
        st["cache"] = []
        for _ in range(2):
            w = torch.randint(-2 ** 31, 2 ** 31 - 1, (B, H, cap, d * bits // 32), generator=g, device=DEV, dtype=torch.int32)
            s = (4.0 / (2 ** bits - 1) * (0.75 + 0.5 * torch.rand((B, H, cap, d // GROUP), generator=g, device=DEV))).to(dt)
            st["cache"].append((w, s, (-2.0 + 0.2 * torch.randn((B, H, cap, d // GROUP), generator=g, device=DEV)).to(dt)))
        st["rows"] = [torch.randn((B, T, H * d), generator=g, device=DEV).to(dt).view(B, T, H, d).transpose(1, 2)
                      for _ in range(2)]
    return st


# ------------------------------------------------------------------ one pass


def _cut(x, case):
    """[rows, V] logits -> the weights sampled from, not normalised, in 64 bits: of the top_k tokens of each row
    (all with 0) those before which less than top_p of their mass lies, in falling order, equal logits by index."""
    x = x.double() / case["temperature"]
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - top)
    if not case["top_k"] and case["top_p"] >= 1.0:
        return w
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(-1, order)
    if case["top_k"]:
        ws[..., case["top_k"]:] = 0.0
    if case["top_p"] < 1.0:
        upto = torch.cumsum(ws, -1)
        before = torch.cat([torch.zeros_like(upto[..., :1]), upto[..., :-1]], -1)
        ws = torch.where(before < case["top_p"] * ws.sum(-1, keepdim=True), ws, 0.0)
    return torch.zeros_like(w).scatter_(-1, order, ws)


def _plain_verify(st, case):
    B, m, V = case["batch"], case["draft"], case["vocab"]
    p = _cut(st["logits"].reshape(-1, V), case)
    p = (p / p.sum(-1, keepdim=True)).reshape(B, m + 1, V)
    u = st["uniforms"].double()
    x = st["draft"].long()
    px = p[:, :m].gather(-1, x[..., None])[..., 0]
    qx = torch.ones_like(px) if st["q"] is None else st["q"].gather(-1, x[..., None])[..., 0].double()
    i = torch.arange(m + 1, device=DEV)
    n_max = torch.full((B,), m, device=DEV) if st["lens"] is None else st["lens"].long()
    ok = (u[:, :m] * qx < px) & (i[:m] < n_max[:, None])
    n = torch.cumprod(ok.long(), -1).sum(-1)
    b = torch.arange(B, device=DEV)
    row = p[b, n]
    if m:
        at = n.clamp(max=m - 1)
        if st["q"] is None:
            taken = torch.zeros_like(row).scatter_(1, x[b, at][:, None], 1.0)
        else:
            taken = st["q"][b, at].double()
        rest = (row - torch.where((n < n_max)[:, None], taken, 0.0)).clamp(min=0.0)
        row = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    cdf = torch.cumsum(row, -1)
    tok = (cdf <= u[:, m:] * cdf[:, -1:]).sum(-1).clamp(max=V - 1)
    drafted = torch.cat([x, x.new_zeros((B, 1))], 1)
    tokens = torch.where(i < n[:, None], drafted, torch.where(i == n[:, None], tok[:, None], -1))
    return n.to(torch.int32), tokens.to(torch.int32), px.float()


def _plain_rope(x, st, case):
    half = case["dims"] // 2
    ang = st["positions"].double()[:, None, :, None] * st["freqs"]              # [B, 1, L, half]
    c, s = torch.cos(ang).float(), torch.sin(ang).float()
    r, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., :half], r[..., half:])
    a, b = a * c - b * s, a * s + b * c
    y = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([y.to(x.dtype), rest], -1)


def _plain_write(trip, rows, at, bits):
    """rows [B, H, T, d] into (words, scales, biases) from position ``at``: scale and bias of every 64 values
    rounded to the cache's type, fields by the rounded ones, each step an operation in 32 bits."""
    words, scales, biases = trip
    B, H, T, d = rows.shape
    levels, per = 2 ** bits - 1, 32 // bits
    x = rows.float().reshape(B, H, T, d // GROUP, GROUP)
    lo = x.amin(-1)
    s, b = ((x.amax(-1) - lo) / levels).to(scales.dtype), lo.to(scales.dtype)
    div = torch.where(s == 0, 1.0, s.float())
    f = torch.round((x - b.float()[..., None]) / div[..., None]).clamp(0, levels).to(torch.int64)
    shift = torch.arange(per, device=DEV) * bits
    w = (f.reshape(B, H, T, d // per, per) << shift).sum(-1)
    words[:, :, at:at + T] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    scales[:, :, at:at + T] = s
    biases[:, :, at:at + T] = b


def _plain_read(trip, upto, bits, dtype):
    w, s, b = (t[:, :, :upto] for t in trip)
    shift = torch.arange(32 // bits, device=DEV, dtype=torch.int32) * bits
    f = ((w[..., None] >> shift) & (2 ** bits - 1)).float().reshape(*s.shape, GROUP)
    return (f * s.float()[..., None] + b.float()[..., None]).reshape(*s.shape[:-1], -1).to(dtype)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "verify":
        if own:
            return _ops().speculative_verify(st["logits"], st["draft"], st["uniforms"], draft_probs=st["q"],
                                             draft_lens=st["lens"], temperature=case["temperature"],
                                             top_k=case["top_k"], top_p=case["top_p"])
        return _plain_verify(st, case)
    if kind == "probs":
        if own:
            return _ops().sampling_probs(st["logits"], temperature=case["temperature"], top_k=case["top_k"],
                                         top_p=case["top_p"])
        w = _cut(st["logits"], case)
        return (w / w.sum(-1, keepdim=True)).float()
    if kind == "rope":
        q, k = st["x"]
        if own:
            return _ops().rope(q, k, st["freqs"], st["positions"], interleaved=case["interleaved"])
        return _plain_rope(q, st, case), _plain_rope(k, st, case)
    bits, at, upto = case["bits"], case["before"], case["before"] + case["rows"]
    keys, values = st["cache"]
    if own:
        ops = _ops()
        ops.quantize_kv(*st["rows"], tuple(t[:, :, at:upto] for t in keys), tuple(t[:, :, at:upto] for t in values),
                        bits=bits)
        return ops.dequantize_kv(tuple(t[:, :, :upto] for t in keys), tuple(t[:, :, :upto] for t in values), bits=bits,
                                 dtype=DTYPES[case["out"]])
    _plain_write(keys, st["rows"][0], at, bits)
    _plain_write(values, st["rows"][1], at, bits)
    return _plain_read(keys, upto, bits, DTYPES[case["out"]]), _plain_read(values, upto, bits, DTYPES[case["out"]])


# ------------------------------------------------------------------ what a pass cannot do without


def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    kind = case["kind"]
    if kind == "verify":
        # the logits once; of the drafter's probabilities a value for every draft and the row of the first one
        # refused (one a sequence); an exponential (8 operations) and a sum for every logit
        B, m, V = case["batch"], case["draft"], case["vocab"]
        q = 4 * B * (m + V) if case["q"] == "dense" and m else 0
        return {"bytes": 2 * B * (m + 1) * V + q + 12 * B * (m + 1), "flops": 9 * B * (m + 1) * V}
    if kind == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n + 4 * n, "flops": 10 * n}
    if kind == "rope":
        rows = case["batch"] * case["rows"]
        heads = case["hq"] + case["hk"]
        return {"bytes": 2 * _size(case["dtype"]) * rows * heads * case["d"] + 8 * rows + 4 * case["dims"],
                "flops": 3 * rows * heads * case["dims"] + 20 * rows * case["dims"]}
    per = 2 * case["batch"] * case["heads"] * case["d"]              # values of a position, keys and values
    upto = case["before"] + case["rows"]
    kept = case["bits"] / 8 + 2 * _size(case["dtype"]) / GROUP       # bytes a value in the cache
    return {"bytes": int(per * (case["rows"] * (2 + kept) + case["before"] * kept + upto * _size(case["out"]))),
            "flops": per * (6 * case["rows"] + 2 * upto)}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits


def _weights_of_row(x, case):
    """numpy float64 logits of one row -> weights with 0 for every token that is cut."""
    w = np.exp((x - x.max()) / case["temperature"])
    k = case["top_k"] or x.size
    if k >= x.size and case["top_p"] >= 1.0:
        return w
    order = np.lexsort((np.arange(x.size), -x))[:k]
    if case["top_p"] < 1.0:
        cum = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[:int(np.searchsorted(cum[:-1], case["top_p"] * cum[-1], side="left"))]
    out = np.zeros_like(w)
    out[order] = w[order]
    return out


def _exact_verify(st, case):
    B, m = case["batch"], case["draft"]
    x = st["logits"].double().cpu().numpy()
    draft = st["draft"].cpu().numpy()
    u = st["uniforms"].double().cpu().numpy()
    lens = np.full(B, m) if st["lens"] is None else st["lens"].cpu().numpy()
    ns, tokens, px = np.zeros(B, np.int32), np.full((B, m + 1), -1, np.int32), np.zeros((B, m))
    for b in range(B):
        stopped = None
        for i in range(m):
            w = _weights_of_row(x[b, i], case)
            p = w / w.sum()
            px[b, i] = p[draft[b, i]]
            if stopped is not None or i >= lens[b]:
                continue
            q = None if st["q"] is None else st["q"][b, i].double().cpu().numpy()
            if u[b, i] * (1.0 if q is None else q[draft[b, i]]) < px[b, i]:
                tokens[b, ns[b]] = draft[b, i]
                ns[b] += 1
                continue
            if q is None:
                q = np.zeros_like(p)
                q[draft[b, i]] = 1.0
            stopped = np.maximum(p - q, 0.0)
            stopped = p if stopped.sum() == 0 else stopped
        if stopped is None:
            stopped = _weights_of_row(x[b, ns[b]], case)
        cdf = np.cumsum(stopped)
        tokens[b, ns[b]] = min(int(np.searchsorted(cdf, u[b, m] * cdf[-1], side="right")), x.shape[-1] - 1)
    return ns, tokens, px


def _exact_kv(st, case):
    bits, at, upto = case["bits"], case["before"], case["before"] + case["rows"]
    r32 = lambda a: a.to(torch.float32).double()        # the definition's steps are operations in 32 bits
    cast = lambda a: a.to(torch.float32).to(DTYPES[case["dtype"]]).double()
    outs = []
    for (w, s, b), rows in zip(st["cache"], st["rows"]):
        B, H, T, d = rows.shape
        old = torch.stack([(w[:, :, :at].to(torch.int64) & 0xFFFFFFFF) // 2 ** (bits * j) % 2 ** bits
                           for j in range(32 // bits)], -1).reshape(B, H, at, d // GROUP, GROUP).double()
        x = rows.double().reshape(B, H, T, d // GROUP, GROUP)
        lo, hi = x.min(-1).values, x.max(-1).values
        sn, bn = cast(r32(hi - lo) / (2 ** bits - 1)), cast(lo)
        new = torch.floor(r32(r32(x - bn[..., None]) / torch.where(sn == 0, 1.0, sn)[..., None]) + 0.0)
        frac = r32(r32(x - bn[..., None]) / torch.where(sn == 0, 1.0, sn)[..., None]) - new
        new = new + ((frac > 0.5) | ((frac == 0.5) & (new % 2 != 0)))           # to the nearest, halves to even
        new = new.clamp(0, 2 ** bits - 1)
        f = torch.cat([old, new], 2)
        sc, bi = torch.cat([s[:, :, :at].double(), sn], 2), torch.cat([b[:, :, :at].double(), bn], 2)
        outs.append((f * sc[..., None] + bi[..., None]).reshape(B, H, upto, d).cpu().numpy())
    return tuple(outs)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "verify":
        return _exact_verify(st, case)
    if kind == "probs":
        ws = [_weights_of_row(x, case) for x in st["logits"].double().cpu().numpy()]
        return np.stack([w / w.sum() for w in ws])
    if kind == "rope":
        # each pair as a complex number, turned by exp(i * position * frequency)
        half, d = case["dims"] // 2, case["d"]
        pos = st["positions"].cpu().numpy().astype(np.float64)
        turn = np.exp(1j * (pos[:, None, :, None] * st["freqs"].cpu().numpy()))
        first = np.arange(half) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        outs = []
        for t in st["x"]:
            v = t.double().cpu().numpy()
            z = (v[..., first] + 1j * v[..., second]) * turn
            y = v.copy()
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    return _exact_kv(st, case)
