"""GPU: ops.token_logprobs against 64 bits.

e^z is off by z 2^-23 (its exponent, rounded twice) and 2^-22 of itself; a lane adds V / 256 of them in fp32, some 64 more sums
join the lanes: S, relative, by less than E = 2^-22 (V / 1024 + 20 + mean |z|), the mean under p; U / S by that of |U / S| more. ln S
is that off, absolutely, and what is given rounds once to fp32 from 64 bits. Alternatives and their order are exact."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(x, tokens, got, top, temperature=1.0):
    given, entropy, ids, best = (t.cpu().numpy() for t in got)
    V = x.shape[-1]
    x = x.reshape(-1, V).double().cpu().numpy()
    tokens = tokens.reshape(-1).cpu().numpy()
    for i in range(x.shape[0]):
        lp, h, order, lps = paged_ref.logprobs(x[i], int(tokens[i]), top, temperature)
        e = 2.0 ** -22 * (V / 1024 + 20 + h)
        close = lambda a, b: a == b or abs(a - b) <= e + abs(b) * 2.0 ** -24
        assert close(given.reshape(-1)[i], lp), (i, given.reshape(-1)[i], lp)
        assert abs(entropy.reshape(-1)[i] - h) <= 2 * e * (1 + h), (i, entropy.reshape(-1)[i], h)
        if top:
            np.testing.assert_array_equal(ids.reshape(-1, top)[i], order)
            assert all(close(a, b) for a, b in zip(best.reshape(-1, top)[i], lps))


def logits(g, rows, V, dtype, dev, spread=2.0):
    x = torch.randn(rows, V, generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (rows, 8), generator=g), 6 * torch.rand(rows, 8, generator=g))
    return x.to(DT[dtype]).to(dev)


def run(x, top, temperature=1.0, seed=0, **kw):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, x.shape[-1], x.shape[:-1], generator=g).to(x.device)
    got = ops.token_logprobs(x, tokens, top=top, temperature=temperature, **kw)
    assert got[0].shape == tokens.shape and got[2].shape == (*tokens.shape, top) and got[2].dtype == torch.int32
    check(x, tokens, got, top, temperature)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 7), (3, 64), (5, 257), (1, 2049), (2, 8192), (3, 20001), (1, 151936), (2, 131073), (700, 515), (530, 9001)])
def test_rows(dev, rows, V, dtype):
    g = torch.Generator().manual_seed(rows + V)
    x = logits(g, rows, V, dtype, dev)
    for top in sorted({0, 1, min(V, 5), min(V, 64)}):
        run(x[:40] if rows > 40 and top > 5 else x, top, temperature=(1.0, 0.6)[top % 2], seed=top)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_equal_rising_and_falling_logits(dev, rows, top, dtype):
    """All equal, two values, rising, falling, the best in one lane's values, all but a few forbidden, nothing at all."""
    V = 9000
    i = torch.arange(V, dtype=torch.float32)
    neg = torch.full((V,), float("-inf"))
    some = neg.clone()
    some[[17, 8999, 4000]] = torch.tensor([1.0, 2.0, 1.0])
    lane = torch.zeros(V)
    lane[4096:4224] = torch.arange(128.0) / 16
    lowest = torch.full((V,), torch.finfo(DT[dtype]).min)
    low_but_one = lowest.clone()
    low_but_one[77] = 3.0
    cases = [torch.zeros(V), -0.0 * i, (i % 2), i / 100, -i / 100, lane, some, neg, torch.full((V,), float("nan")), lowest, low_but_one,
             torch.where(i % 3 == 0, neg, i % 50), i - 5000]
    x = torch.stack(cases).to(DT[dtype]).to(dev)
    if rows > 1:
        x = x.repeat(rows // len(cases), 1)
    n = min(x.shape[0], len(cases))
    from dspark_rocm import ops

    tokens = torch.randint(0, V, (x.shape[0],), generator=torch.Generator().manual_seed(top)).to(dev)
    got = ops.token_logprobs(x, tokens, top=top)
    check(x[:n], tokens[:n], [t[:n] for t in got], top)
    for t in got[1:]:                           # a row's numbers do not depend on its neighbours
        for r in range(n, x.shape[0], n):
            m = min(n, x.shape[0] - r)
            assert torch.equal(t[r:r + m], t[:m])


def test_infinite_and_nan_logits(dev):
    g = torch.Generator().manual_seed(1)
    for V in (100, 30000):
        x = logits(g, 4, V, "bf16", dev)
        x[0, 5] = x[0, V - 1] = x[1, 7] = float("inf")
        x[2, ::2] = float("nan")
        x[3, 1:] = float("nan")
        x[3, 0] = float("-inf")
        from dspark_rocm import ops

        for tokens in (torch.tensor([5, 7, 1, 0]), torch.tensor([4, 4, 2, 5]), torch.tensor([-1, V, 2 ** 40, -2 ** 40])):
            tokens = tokens.to(dev)
            check(x, tokens, ops.token_logprobs(x, tokens, top=9), 9)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [2559, 2560, 2561, 5121, 163839, 163841])
def test_rows_that_end_where_a_step_does(dev, V, dtype):
    """A wave of a split row takes 2560 values a step; rows at every offset from 16 bytes reach one load further."""
    g = torch.Generator().manual_seed(V)
    wide = logits(g, 2, V + 9, dtype, dev)
    for off in (0, 1, 7):
        run(wide[:, off:off + V], 20, seed=off)


def test_views_streams_and_workspaces(dev):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(2)
    wide = logits(g, 6, 20011, "bf16", dev)
    for x in (wide[:, 3:20003], wide[::2], wide.t()[:700].t(), wide.view(2, 3, 20011), wide[0], wide[1:2].expand(4, 20011)):
        tokens = torch.randint(0, x.shape[-1], x.shape[:-1], generator=g).to(dev)
        ws = torch.full((ops.token_logprobs_workspace_bytes(max(tokens.numel(), 1), x.shape[-1], 7),), 255, dtype=torch.uint8, device=dev)
        want = ops.token_logprobs(x, tokens, top=7)
        check(x, tokens, want, 7)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = ops.token_logprobs(x, tokens.to(torch.int32), top=7, workspace=ws)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured(dev):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(3)
    x, tokens = logits(g, 3, 50257, "f16", dev), torch.tensor([1, 2, 3], device=dev, dtype=torch.int32)
    call = lambda: ops.token_logprobs(x, tokens, top=20)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        x.copy_(logits(g, 3, 50257, "f16", dev))
        tokens += 11
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_past_32_bits(dev):
    from dspark_rocm import ops

    V = 4000
    buf = torch.zeros((1 << 32) + V + 9, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(4)
    x = logits(g, 3, V, "bf16", dev)
    view = buf.as_strided((3, V), ((1 << 31) + 3, 1))
    view.copy_(x)
    tokens = torch.tensor([1, 2, 3], device=dev)
    got, want = ops.token_logprobs(view, tokens, top=5), ops.token_logprobs(x, tokens, top=5)
    for a, b in zip(got, want):
        assert torch.equal(a, b) if a.dtype == torch.int32 else torch.allclose(a, b, rtol=0, atol=1e-5)


def test_with_a_sampled_round(dev):
    """What a served token is reported with, beside the operators that chose it: its probability is the sampler's."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(5)
    x = logits(g, 4, 32003, "bf16", dev).view(1, 4, -1)
    draft = torch.randint(0, 32003, (1, 3), generator=g).to(dev)
    n, tokens, px = ops.speculative_verify(x, draft, torch.rand(1, 4, generator=g).to(dev))
    lp, h, ids, best = ops.token_logprobs(x[:, :3], draft, top=3)
    assert torch.allclose(lp.exp(), px, rtol=1e-5, atol=0)
    p = ops.sampling_probs(x[:, :3])
    assert torch.equal(p.argmax(-1).int(), ids[..., 0]) and torch.allclose(p.gather(-1, ids.long()), best.exp(), rtol=1e-5, atol=0)
