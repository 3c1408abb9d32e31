"""GPU: sampling_probs and speculative_verify against the oracle in 64 bits.

Counts and tokens are equal. A probability is one fp64 value rounded to fp32: half a step of it (2^-24)
beside the fp64 error of two weights (5e-15 of the polynomial, |argument| 2^-53 <= 1.2e-13 each) and sums."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sampling_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _np(t):
    return t.detach().double().cpu().numpy()


def close(got, want):
    got, want = _np(got), np.asarray(want)
    assert got.shape == want.shape
    assert (np.abs(got - want) <= want * (2.0 ** -24 + 1e-12) + 2.0 ** -150).all(), np.abs(got - want).max()


def rows(g, n, V, dtype, kind="plain"):
    x = 3.0 * torch.randn(n, V, generator=g)
    if kind == "ties":
        x = torch.round(x)
    elif kind == "same":
        x = torch.full((n, V), -1.25)
    elif kind == "masked":                               # most of the row cut off, as a grammar does; type's lowest too
        x = torch.where(torch.rand(n, V, generator=g) < 0.97, float("-inf"), x)
        x[:, ::7] = torch.finfo(dtype).min
        x[:, V // 2] = 0.5
    elif kind == "zeros":                                # +0 and -0 are equal logits
        x = torch.where(torch.rand(n, V, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "odd":                                  # values that are not finite
        x[:, ::5] = float("nan")
        x[:, 1::5] = float("-inf")
        if n > 1:
            x[1, V // 3] = x[1, -1] = float("inf")
        if n > 2:
            x[2] = float("-inf")
        if n > 3:
            x[3] = float("nan")
    elif kind == "far":                                  # the whole range of the type, tiny values among them
        x = x * torch.exp2(torch.randint(-20, 4, (n, V), generator=g).float())
    return x.to(dtype)


CUTS = [dict(), dict(top_k=1), dict(top_k=20), dict(top_p=0.9), dict(top_k=50, top_p=0.8), dict(top_p=1e-9),
        dict(temperature=0.25, top_p=0.999), dict(temperature=3.0, top_k=700)]


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "masked", "zeros", "odd", "far"])
@pytest.mark.parametrize("n,V,dtype", [(4, 1, "bf16"), (4, 7, "f16"), (4, 511, "bf16"), (4, 513, "f16"), (4, 5000, "bf16"),
                                       (5, 50257, "f16"), (4, 151936, "bf16")])
def test_probs(dev, n, V, dtype, kind):
    from dspark_rocm import ops

    x = rows(torch.Generator().manual_seed(V + n), n, V, DT[dtype], kind)
    for kw in CUTS:
        got = ops.sampling_probs(x.to(dev), **kw)
        assert got.dtype == torch.float32
        close(got, np.stack([ref.probs(r, **kw) for r in _np(x)]))


def test_probs_of_the_longest_row(dev):
    from dspark_rocm import ops

    x = rows(torch.Generator().manual_seed(0), 1, 524280, torch.bfloat16)
    for kw in (dict(), dict(top_p=0.97), dict(top_k=1000, top_p=0.9)):
        close(ops.sampling_probs(x.to(dev), **kw), ref.probs(_np(x)[0], **kw)[None])
    with pytest.raises(ValueError):
        ops.sampling_probs(torch.zeros(1, 524281, dtype=torch.bfloat16, device=dev))


def _drafts(g, x, kind, m):
    """Drafts from a distribution near the target's, and it."""
    B, _, V = x.shape
    q = torch.softmax(torch.nan_to_num(x[:, :m].float(), 0.0, 5.0, -30.0).clamp(-30, 30) + torch.randn(B, m, V, generator=g), -1)
    d = torch.multinomial(q.reshape(-1, V), 1, generator=g).reshape(B, m) if m else torch.zeros(B, 0, dtype=torch.int64)
    return d.to(torch.int32), q


@pytest.mark.parametrize("kind", ["plain", "ties", "masked", "odd"])
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("B,m,V,dtype", [(1, 0, 8192, "bf16"), (3, 1, 1, "bf16"), (2, 4, 9, "f16"), (5, 3, 777, "bf16"),
                                         (1, 15, 32003, "f16"), (7, 2, 4096, "bf16"), (2, 3, 151936, "bf16")])
def test_verify(dev, B, m, V, dtype, kind, dense):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(B * 1000 + m * 10 + V)
    x = rows(g, B * (m + 1), V, DT[dtype], kind).reshape(B, m + 1, V)
    d, q = _drafts(g, x, kind, m)
    seen = set()
    for i, kw in enumerate(CUTS):
        u = torch.rand(B, m + 1, generator=g, dtype=torch.float64 if i % 2 else torch.float32)
        lens = torch.randint(0, m + 1, (B,), generator=g) if i % 3 == 2 else None
        got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev) if dense else None,
                                     draft_lens=None if lens is None else lens.to(dev), **kw)
        want = ref.verify(_np(x), d.numpy(), u.numpy(), q.numpy() if dense else None, None if lens is None else lens.numpy(), **kw)
        assert np.array_equal(got[0].cpu().numpy(), want[0]), (kw, got[0], want[0])
        assert np.array_equal(got[1].cpu().numpy(), want[1]), (kw, got[1], want[1])
        close(got[2], want[2])
        seen.update(want[0].tolist())
    assert len(seen) > 1 or not (dense and kind == "plain" and m > 1 and V > 9)     # drafts are taken and refused


def test_verify_takes_what_the_reference_would_index(dev):
    """Drafts outside the vocabulary, lengths outside the batch, random numbers at and past both ends, the same
    token drafted twice, int64 drafts: refused, clamped or drawn, and nothing read out of range."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(5)
    x = rows(g, 12, 1000, torch.bfloat16).reshape(3, 4, 1000)
    best = x.float().argmax(-1)[:, :3]
    for d in (torch.tensor([[-1, 5, 5]] * 3), torch.tensor([[1000, 0, 0]] * 3), torch.tensor([[2 ** 31 - 1, 0, 0]] * 3),
              torch.tensor([[2 ** 32 + 7, 0, 0]] * 3), best):
        for u in (torch.zeros(3, 4), torch.full((3, 4), 1.0 - 2.0 ** -24), torch.full((3, 4), 1.0), torch.full((3, 4), 2.0)):
            for lens in (None, torch.tensor([-4, 1, 99])):
                for dense in (False, True):
                    q = torch.softmax(x[:, :3].float(), -1)
                    for kw in (dict(), dict(top_k=5)):
                        got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev) if dense else None,
                                                     draft_lens=None if lens is None else lens.to(dev), **kw)
                        want = ref.verify(_np(x), d.clamp(-1, 2 ** 31 - 1).numpy(), u.numpy(), q.numpy() if dense else None,
                                          None if lens is None else lens.numpy(), **kw)
                        assert np.array_equal(got[0].cpu().numpy(), want[0])
                        if dense and not kw:
                            continue        # p = q but for their roundings: the rest is the roundings' own pattern
                        assert np.array_equal(got[1].cpu().numpy(), want[1])


@pytest.mark.parametrize("cut", [dict(), dict(top_k=30, top_p=0.9)])
def test_views_and_strides(dev, cut):
    """Rows at any address and stride: a column slice from an odd column, sequences and rows exchanged, a
    transposed vocabulary, expanded logits; draft probabilities a slice too."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(9)
    big = rows(g, 20, 3001, torch.bfloat16).reshape(4, 5, 3001).to(dev)
    u = torch.rand(5, 4, generator=g).to(dev)
    for x in (big[:, :, 3:2999].transpose(0, 1), big[:, :, :1001].transpose(0, 1),
              big.transpose(1, 2).contiguous().transpose(1, 2).transpose(0, 1), big[:1].expand(4, 5, 3001).transpose(0, 1)):
        V = x.shape[2]
        d, q = _drafts(g, x.cpu(), "plain", 3)
        wide = torch.zeros(5, 3, V + 3, device=dev)
        wide[:, :, 1:V + 1] = q.to(dev)
        got = ops.speculative_verify(x, d.to(dev), u, draft_probs=wide[:, :, 1:V + 1], **cut)
        want = ref.verify(_np(x), d.numpy(), _np(u), q.numpy(), **cut)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
        close(got[2], want[2])
        close(ops.sampling_probs(x[:, 0], **cut), np.stack([ref.probs(r, **cut) for r in _np(x[:, 0])]))


def test_out_and_workspace(dev):
    """out is written and nothing beside it; a workspace of any content serves, one too small or misplaced does not."""
    from dspark_rocm import ops

    x = rows(torch.Generator().manual_seed(2), 3, 1003, torch.float16).to(dev)
    buf = torch.full((3 * 1003 + 2,), 7.0, device=dev)
    out = buf[1:-1].view(3, 1003)
    need = ops.sampling_workspace_bytes(3, 1003)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)
    for kw in CUTS:
        assert ops.sampling_probs(x, out=out, workspace=ws, **kw) is out
        close(out, np.stack([ref.probs(r, **kw) for r in _np(x)]))
        assert buf[0] == 7 and buf[-1] == 7
    for bad in (dict(workspace=ws[:-1]), dict(workspace=ws.cpu()), dict(out=out.t()), dict(out=out.half()), dict(out=out[:2])):
        with pytest.raises(ValueError):
            ops.sampling_probs(x, **bad)


def test_refusals(dev):
    from dspark_rocm import ops

    x = torch.zeros(2, 3, 10, dtype=torch.bfloat16, device=dev)
    d, u = torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.zeros(2, 3, device=dev)
    for bad in (dict(draft_probs=torch.zeros(2, 2, 9, device=dev)), dict(draft_probs=torch.zeros(2, 2, 10, device=dev).half()),
                dict(draft_lens=torch.zeros(3, dtype=torch.int32, device=dev)), dict(draft_lens=torch.zeros(2, device=dev)),
                dict(draft_probs=torch.zeros(2, 2, 10)), dict(temperature=0.0), dict(top_p=0.0),
                dict(draft_probs=torch.zeros(2, 2, 10, device=dev, requires_grad=True))):
        with pytest.raises(ValueError):
            ops.speculative_verify(x, d, u, **bad)
    for args in ((x[0], d, u), (x, d[:, :1], u), (x, d.float(), u), (x, d, u[:, :2]), (x, d, u.half()), (x, d.cpu(), u)):
        with pytest.raises(ValueError):
            ops.speculative_verify(*args)
    for f in (lambda: ops.speculative_verify(x.float(), d, u), lambda: ops.sampling_probs(x.float())):
        with pytest.raises(TypeError):
            f()
    assert ops.sampling_probs(x[:0]).shape == (0, 3, 10)
    assert [tuple(t.shape) for t in ops.speculative_verify(x[:0], d[:0], u[:0])] == [(0,), (0, 3), (0, 2)]


@pytest.mark.parametrize("cut", [dict(), dict(top_k=20, top_p=0.9)])
def test_streams_and_graphs(dev, cut):
    """On another stream; two captured graphs replayed in turn with the program's own calls between."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(4)
    sets = []
    for _ in range(2):
        x = rows(g, 8, 20000, torch.bfloat16).reshape(2, 4, 20000)
        d, q = _drafts(g, x, "plain", 3)
        sets.append([t.to(dev) for t in (x, d, torch.rand(2, 4, generator=g), q)])
    call = lambda s: ops.speculative_verify(s[0], s[1], s[2], draft_probs=s[3], **cut)
    want = [[t.clone() for t in call(s)] for s in sets]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        outs = [call(s) for s in sets]
    other.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call(s)
        graphs.append((graph, o))
    for _ in range(3):
        for (graph, o), w in zip(graphs, want):
            for t in o:
                t.zero_()
            graph.replay()
            call(sets[0])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(w, o))
    sets[0][2].copy_(torch.rand(2, 4, generator=g))         # new random numbers in place, as a serving loop draws them
    graphs[0][0].replay()
    assert all(torch.equal(a, b) for a, b in zip(call(sets[0]), graphs[0][1]))


@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_many_rows_uncut(dev, temperature):
    """A batch large enough for its weights to come from a table of the values: plain rows, values near 0, beyond
    256 and below -256 (all of a row, and beside others), infinities, NaN, rows that leave nothing."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(6)
    n, V = 60, 151931
    x = 3.0 * torch.randn(n, V, generator=g)
    x[1] = x[1] * torch.exp2(torch.randint(-140, 2, (V,), generator=g).float())
    x[2] = x[2] * 200
    x[3] = x[3] - 300
    x[4] -= 200
    x[5, ::2] = torch.finfo(torch.bfloat16).min
    x[6] = float("-inf")
    x[7] = float("nan")
    x[8, ::3], x[8, 1::3] = float("nan"), float("-inf")
    x[9, 77] = x[9, 100000] = float("inf")
    x[10] = 0.0
    x[11, ::2], x[11, 1::2] = -0.0, -256.0
    x[12] = 255.0 + x[12]
    x[13] = -1e-30
    x = x.to(torch.bfloat16)
    want = [ref.probs(r, temperature=temperature) for r in _np(x)]
    got = ops.sampling_probs(x.to(dev), temperature=temperature)
    close(got, np.stack(want))
    d, q = _drafts(g, x.view(15, 4, V), "plain", 3)
    u = torch.rand(15, 4, generator=g)
    got = ops.speculative_verify(x.view(15, 4, V).to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev), temperature=temperature)
    ns, tokens, px = ref.verify(_np(x).reshape(15, 4, V), d.numpy(), u.numpy(), q.numpy(), temperature=temperature)
    assert np.array_equal(got[0].cpu().numpy(), ns) and np.array_equal(got[1].cpu().numpy(), tokens)
    close(got[2], px)


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_p=0.5, temperature=2.0), dict(top_k=400), dict(top_k=500, top_p=0.7)])
@pytest.mark.parametrize("n,V,dtype", [(100, 20000, "bf16"), (30, 60000, "f16"), (200, 3000, "f16"), (3, 400001, "bf16")])
def test_many_candidates(dev, n, V, dtype, kw):
    """Rows counted by several workgroups each, and more rows than that: wide and tied values, a row of one value,
    one with too many distinct values for one pass."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(n)
    x = torch.cat([rows(g, n - 3, V, DT[dtype]), rows(g, 1, V, DT[dtype], "same"), rows(g, 1, V, DT[dtype], "far"),
                   rows(g, 1, V, DT[dtype], "ties")]) if n > 3 else rows(g, n, V, DT[dtype], "ties")
    close(ops.sampling_probs(x.to(dev), **kw), np.stack([ref.probs(r, **kw) for r in _np(x)]))
    m = 2 if n % 3 == 0 else 1
    x = x[:n // (m + 1) * (m + 1)].view(-1, m + 1, V)
    d, q = _drafts(g, x, "plain", m)
    u = torch.rand(x.shape[0], m + 1, generator=g)
    for dense in (False, True):
        got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev) if dense else None, **kw)
        ns, tokens, px = ref.verify(_np(x), d.numpy(), u.numpy(), q.numpy() if dense else None, **kw)
        assert np.array_equal(got[0].cpu().numpy(), ns) and np.array_equal(got[1].cpu().numpy(), tokens)
        close(got[2], px)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.8), dict(top_k=130, top_p=0.9)])
def test_many_short_rows_and_long_blocks(dev, kw):
    """The most rows and the most drafts a call takes; one more of either is refused."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(8)
    x = rows(g, 60000, 40, torch.bfloat16).view(30000, 2, 40)
    d, q = _drafts(g, x, "plain", 1)
    u = torch.rand(30000, 2, generator=g)
    got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev), **kw)
    pick = slice(0, 30000, 37)
    n, tokens, px = ref.verify(_np(x[pick]), d[pick].numpy(), u[pick].numpy(), q[pick].numpy(), **kw)
    assert np.array_equal(got[0][pick].cpu().numpy(), n) and np.array_equal(got[1][pick].cpu().numpy(), tokens)
    close(got[2][pick], px)
    close(ops.sampling_probs(x[pick].to(dev), **kw), np.stack([[ref.probs(r, **kw) for r in s] for s in _np(x[pick])]))
    x = rows(g, 512, 3000, torch.float16).view(2, 256, 3000)
    x[:, :, 7] = 30.0
    d = torch.full((2, 255), 7)
    d[1, 200] = 8
    u = torch.rand(2, 256, generator=g)
    got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), **kw)
    n, tokens, px = ref.verify(_np(x), d.numpy(), u.numpy(), **kw)
    assert n[0] > 200 and np.array_equal(got[0].cpu().numpy(), n) and np.array_equal(got[1].cpu().numpy(), tokens)
    close(got[2], px)
    with pytest.raises(ValueError):
        ops.speculative_verify(x[:, :1].expand(2, 257, 3000).to(dev), d[:, :1].expand(2, 256).to(dev), torch.rand(2, 257, device=dev))
    with pytest.raises(ValueError):
        ops.sampling_probs(torch.zeros(65536, 2, dtype=torch.bfloat16, device=dev))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(top_p=0.9)])
def test_the_same_bits_each_time(dev, kw):
    """Repeated calls on one input, with other calls between on another stream: nothing depends on which workgroup
    arrives last."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(12)
    x = rows(g, 24, 100003, torch.bfloat16, "ties").view(4, 6, 100003)
    d, q = _drafts(g, x, "plain", 5)
    args = x.to(dev), d.to(dev), torch.rand(4, 6, generator=g).to(dev)
    q = q.to(dev)
    want = ops.speculative_verify(*args, draft_probs=q, **kw)
    probs = ops.sampling_probs(args[0], **kw)
    other = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(other):
            ops.sampling_probs(args[0], **kw)
        got = ops.speculative_verify(*args, draft_probs=q, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(ops.sampling_probs(args[0], **kw), probs)
    torch.cuda.synchronize()


@pytest.mark.parametrize("top_p", [1.0, 0.85])
@pytest.mark.parametrize("top_k", [1, 31, 64, 65, 128, 129])
@pytest.mark.parametrize("V,dtype", [(600, "bf16"), (40961, "f16"), (70001, "bf16"), (140000, "bf16")])
def test_tied_candidates(dev, V, dtype, top_k, top_p):
    """Rows of which more tokens tie for the top_k than are looked at one by one, and rows without ties whose
    candidates are about as many: the first by index count, over every segment."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(V + top_k)
    B, m = 4, 2
    x = rows(g, B * (m + 1), V, DT[dtype])
    x[0] = 1.5                                           # nothing but ties
    x[1] = torch.round(x[1].float() / 4).to(x.dtype) * 4     # thousands at each value
    x[2, torch.randperm(V, generator=g)[:400]] = 20.0    # more than are sorted, spread, above the others
    x[3, V - 300:] = 9.5                                 # in the last segments
    x[4, :70] = 30.0                                     # some above a tie
    x[4, 70:] = torch.where(torch.rand(V - 70, generator=g) < 0.5, -2.0, -3.0).to(x.dtype)
    x[5] = float("-inf")
    x[5, ::2] = float("nan")
    x[5, 100:400] = -1.0
    x = x.reshape(B, m + 1, V)
    d, q = _drafts(g, x, "odd", m)
    u = torch.rand(B, m + 1, generator=g, dtype=torch.float64)
    for qq in (None, q):
        got = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=None if qq is None else qq.to(dev),
                                     top_k=top_k, top_p=top_p)
        want = ref.verify(_np(x), d.numpy(), u.numpy(), None if qq is None else qq.numpy(), top_k=top_k, top_p=top_p)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
        close(got[2], want[2])
    flat = x.reshape(-1, V)[:6]
    close(ops.sampling_probs(flat.to(dev), top_k=top_k, top_p=top_p), np.stack([ref.probs(r, top_k=top_k, top_p=top_p) for r in _np(flat)]))


@pytest.mark.parametrize("kw", [dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.9999), dict(top_k=9000, top_p=0.999), dict(top_k=19990)])
@pytest.mark.parametrize("n", [2, 300])
@pytest.mark.parametrize("dtype,t", [("f16", 2e5), ("f16", 3.0), ("bf16", 1e30), ("bf16", 1.0)])
def test_every_value_of_the_type(dev, dtype, t, n, kw):
    """Logits of any finite bits at a temperature of the type's range: the cut lies thousands of values below the
    largest, past what is counted at a time, near and below zero."""
    from dspark_rocm import ops

    V = 20000
    g = torch.Generator().manual_seed(n)
    x = torch.randint(-2 ** 15, 2 ** 15, (n, V), generator=g, dtype=torch.int32).to(torch.int16).view(DT[dtype])
    x = torch.where(torch.isfinite(x), x, 0.0)
    got = ops.sampling_probs(x.to(dev), temperature=t, **kw)
    pick = range(n) if n < 10 else range(0, n, 61)
    close(got[list(pick)], np.stack([ref.probs(r, temperature=t, **kw) for r in _np(x[list(pick)])]))


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "masked", "odd", "far"])
@pytest.mark.parametrize("V,dtype", [(1, "bf16"), (9, "f16"), (513, "bf16"), (8192, "f16"), (50257, "bf16"), (81905, "bf16"),
                                     (81913, "f16"), (81920, "bf16"), (100001, "f16")])
def test_rows_without_drafts(dev, V, dtype, kind):
    """The next token of each row, sampled; around the length to which a row is taken whole."""
    from dspark_rocm import ops

    n = 5
    g = torch.Generator().manual_seed(V)
    x = rows(g, n, V, DT[dtype], kind).reshape(n, 1, V)
    none = torch.zeros(n, 0, dtype=torch.int32, device=dev)
    for kw in (dict(top_k=1), dict(top_k=20, top_p=0.9), dict(top_k=128), dict(top_k=100, top_p=0.7, temperature=0.5)):
        u = torch.rand(n, 1, generator=g, dtype=torch.float64)
        got = ops.speculative_verify(x.to(dev), none, u.to(dev), **kw)
        want = ref.verify(_np(x), np.zeros((n, 0), np.int32), u.numpy(), None, None, **kw)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1]), (kw, got, want)
        buf = torch.full((n * V + 8,), 7.0, device=dev)
        out = buf[3:3 + n * V].view(n, 1, V)
        close(ops.sampling_probs(x.to(dev), out=out, **kw)[:, 0], np.stack([ref.probs(r, **kw) for r in _np(x[:, 0])]))
        assert (buf[:3] == 7).all() and (buf[3 + n * V:] == 7).all()


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.8), dict(top_k=300)])
def test_offsets_past_32_bits(dev, kw):
    """Sequences and rows whose logits and draft probabilities lie more than 2^31 elements apart."""
    from dspark_rocm import ops

    V, far = 5001, (1 << 31) + 17
    g = torch.Generator().manual_seed(3)
    x = rows(g, 4, V, torch.bfloat16).reshape(2, 2, V)
    d, q = _drafts(g, x, "plain", 1)
    u = torch.rand(2, 2, generator=g, dtype=torch.float64)
    want = ops.speculative_verify(x.to(dev), d.to(dev), u.to(dev), draft_probs=q.to(dev), **kw)
    buf, qbuf = torch.empty(far + 2 * V, dtype=torch.bfloat16, device=dev), torch.empty(far + 2 * V, device=dev)
    qs = qbuf.as_strided((2, 1, V), (far, V, 1)).copy_(q)
    for strides in ((far, V, 1), (V, far, 1)):
        xs = buf.as_strided((2, 2, V), strides).copy_(x)
        got = ops.speculative_verify(xs, d.to(dev), u.to(dev), draft_probs=qs, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs = buf.as_strided((2, V), (far, 1)).copy_(x[:, 0])
    assert torch.equal(ops.sampling_probs(xs, **kw), ops.sampling_probs(x[:, 0].contiguous().to(dev), **kw))
    del buf, qbuf, qs, xs
    torch.cuda.empty_cache()


def test_border_of_two_tokens(dev):
    """Rows of two logits x < 0 and 0: the first token weighs w = 2^(x c), and is drawn while u (1 + w) < w. With
    |x c| <= 1/2, w is within 5.2e-16 of itself (3.2e-16 of the interpolation, 1.4e-16 of its steps' roundings, the rest the
    argument's); in u = w / (1 + w) that counts 0.59 times, beside the roundings of 1 + w, u (1 + w) and u (2.2e-16):
    5.3e-16. So random numbers 6e-16 beside the border fall on either side."""
    from dspark_rocm import ops

    x = -torch.arange(0x3C80, 0x3EB1, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    assert float(x.float().min()) > -0.3466
    logits = torch.stack([x, torch.zeros_like(x)], -1)[:, None].to(dev)
    w = np.exp(x.double().numpy().astype(np.longdouble))
    none = torch.zeros(len(x), 0, dtype=torch.int32, device=dev)
    for side, token in ((-1, 0), (1, 1)):
        u = (w / (1 + w) * (1 + side * np.longdouble(6e-16))).astype(np.float64)
        got = ops.speculative_verify(logits, none, torch.from_numpy(u)[:, None].to(dev))[1]
        assert (got == token).all(), int((got != token).sum())


@pytest.mark.parametrize("kw", CUTS + [dict(top_k=128, top_p=0.9), dict(top_k=129), dict(top_k=10 ** 6)])
def test_a_workspace_for_the_sampler(dev, kw):
    """As much as its sampler needs, between guards that stay as they were: the results of a workspace for any."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(11)
    B, m, V = 5, 3, 50257
    x = rows(g, B * (m + 1), V, torch.bfloat16).view(B, m + 1, V)
    d, q = _drafts(g, x, "plain", m)
    args = x.to(dev), d.to(dev), torch.rand(B, m + 1, generator=g).to(dev)
    q, k, p = q.to(dev), kw.get("top_k", 0), kw.get("top_p", 1.0)
    calls = [(0, lambda ws: (ops.sampling_probs(args[0].view(-1, V), workspace=ws, **kw),)),
             (B, lambda ws: ops.speculative_verify(*args, draft_probs=q, workspace=ws, **kw)),
             (B, lambda ws: ops.speculative_verify(*args, workspace=ws, **kw))]
    for seqs, call in calls:
        need, most = (ops.sampling_workspace_bytes(B * (m + 1), V, seqs, *s) for s in ((k, p), ()))
        want = call(torch.full((most,), 0xFF, dtype=torch.uint8, device=dev))
        buf = torch.full((need + 512,), 0xA5, dtype=torch.uint8, device=dev)
        got = call(buf[256:256 + need])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (buf[:256] == 0xA5).all() and (buf[256 + need:] == 0xA5).all()
        with pytest.raises(ValueError):
            call(buf[256:255 + need])
