"""GPU: the operators together as a target runs them: rounds at a temperature, and targets whose rotation goes
by a frequency table, over plain and quantized caches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _model_util import tiny_model
from oracle import sampling_ref as ref

pytestmark = pytest.mark.gpu

SCALED = [dict(rope_scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64)),
          dict(rope_traditional=True), dict(rope_dims=32, rope_scaling=dict(type="linear", factor=2.0))]


def _target(dev, kv_bits=None, **kw):
    from dspark_rocm.model import Target

    return Target(tiny_model(dev, **kw), kv_bits=kv_bits)


def _rows(cache):
    out = []
    for c in cache:
        for part in c.fetch():
            out += [p.clone() for p in part] if isinstance(part, tuple) else [part.clone()]
    return out


@pytest.mark.parametrize("kw", [dict(temperature=0.8, top_k=40, top_p=0.9), dict(temperature=1.2), dict(top_p=0.5)])
@pytest.mark.parametrize("kv_bits,rope", [(None, {}), (8, {}), (4, SCALED[0]), (None, SCALED[2])])
def test_rounds_follow_the_rule(dev, kv_bits, rope, kw):
    """Each round's tokens are the oracle's on the logits of the same verify, its cache the accepted rows."""
    from dspark_rocm import ops

    tgt = _target(dev, kv_bits, **rope)
    cache, mirror = tgt.make_cache(8), tgt.make_cache(8)
    g = torch.Generator().manual_seed(1)
    pending, taken = 3, set()
    for m in (0, 5, 15, 1, 7):
        # a drafter that knows the target's distribution up to an error, and its own probabilities
        probe, _ = tgt.verify(torch.randint(0, 512, (1, m + 1), generator=g), mirror)
        tgt.rollback(mirror, m + 1)
        q = ops.sampling_probs(probe[0, :m].clone(), **kw) if m % 2 else None
        draft = torch.randint(0, 512, (m,), generator=g).tolist() if q is None else \
            torch.multinomial(q.cpu(), 1, generator=g)[:, 0].tolist()
        u = torch.rand(m + 1, generator=g)
        offset = cache[0].offset
        logits, _ = tgt.verify(torch.tensor([[pending] + draft]), mirror)
        want = ref.verify(logits.double().cpu().numpy(), np.array([draft], np.int64).reshape(1, m), u[None].numpy(),
                          None if q is None else q[None].cpu().numpy(), **kw)
        n = int(want[0][0])
        tgt.rollback(mirror, m - n)
        got_n, tokens, ctx = tgt.sampled_round(pending, draft, cache, (0, 1), draft_probs=q, uniforms=u, **kw)
        assert (got_n, tokens) == (n, [int(t) for t in want[1][0] if t >= 0])
        assert cache[0].offset == offset + n + 1 and ctx.shape == (1, n + 1, 512)
        assert all(torch.equal(a, b) for a, b in zip(_rows(cache), _rows(mirror)))
        pending = tokens[-1]
        taken.add(n)
    a = tgt.sampled_round(pending, [1, 2], cache, generator=torch.Generator(device=dev).manual_seed(7), **kw)[:2]
    tgt.rollback(cache, a[0] + 1)
    assert a == tgt.sampled_round(pending, [1, 2], cache, generator=torch.Generator(device=dev).manual_seed(7), **kw)[:2]


def test_top_1_is_the_greedy_round(dev):
    tgt = _target(dev)
    a, b = tgt.make_cache(8), tgt.make_cache(8)
    g = torch.Generator().manual_seed(2)
    p = 5
    for m in (3, 0, 15):
        first = [int(tgt.greedy_round(p, [], a)[1][0])]
        tgt.rollback(a, 1)
        draft = (first + torch.randint(0, 512, (m,), generator=g).tolist())[:m]
        want = tgt.greedy_round(p, draft, a)
        got = tgt.sampled_round(p, draft, b, top_k=1, temperature=0.5)
        assert got[:2] == want[:2] and (m == 0 or got[0] >= 1)
        p = want[1][-1]


def test_round_refusals(dev):
    """Refused before the caches take a row."""
    tgt = _target(dev)
    cache = tgt.make_cache(8)
    for draft, kw in (([1, 2], dict(temperature=0.0)), ([1, 2], dict(top_p=0.0)), ([1, 2], dict(uniforms=torch.rand(2))),
                      ([1, 512], {}), ([-1], {}), ([1] * 16, {}), ([1], dict(draft_probs=torch.zeros(1, 511, device=dev))),
                      ([1], dict(draft_probs=torch.zeros(1, 512, device=dev).half())),
                      ([1], dict(draft_probs=torch.zeros(1, 512, device=dev, requires_grad=True)))):
        with pytest.raises(ValueError):
            tgt.sampled_round(3, draft, cache, **kw)
        assert cache[0].offset == 0


@pytest.mark.parametrize("kv_bits", [None, 8, 4])
@pytest.mark.parametrize("rope", SCALED)
def test_table_targets_step_as_their_module_path(dev, rope, kv_bits):
    """Prefill rows, a verify block and a captured step: the engine against the module path (torch norms and
    attention between the same rotations), apart from the target without the table."""
    from dspark_rocm.model import Target

    tgt, plain = _target(dev, kv_bits, **rope), _target(dev, kv_bits)
    ids = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(3)).to(dev)
    caches = [t.make_cache(128) for t in (tgt, tgt, plain)]
    got, want, other = [], [], []
    for lo, hi in ((0, 40), (40, 44), (44, 60)):
        step = ids[:, lo:hi]
        if hi - lo > 16:
            for t, c in zip((tgt, tgt, plain), caches):
                t.prefill(step, c)
            continue
        got.append(tgt.verify(step, caches[0])[0].clone())
        want.append(tgt.model(step, caches[1]))
        other.append(plain.verify(step, caches[2])[0].clone())
    far = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    for a, b, c in zip(got, want, other):
        assert far(a, b) <= 2.0 ** -6 and far(c, b) > 2.0 ** -4
    e, c = tgt.engine, caches[0]
    graph = torch.cuda.CUDAGraph()
    tgt.rollback(c, 16)
    e.ids[:16].copy_(ids[0, 44:])
    with torch.cuda.graph(graph):
        e.step(16, c, 44)
    for _ in range(3):
        e.logits.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(e.logits, got[-1][0])


def test_round_takes_uniforms_of_any_strides(dev):
    """Random numbers that lie in memory in another order than they count in: read in theirs, and the caches advance by
    the accepted rows."""
    tgt = _target(dev)
    draft = torch.randint(0, 512, (15,), generator=torch.Generator().manual_seed(4)).tolist()
    u = torch.rand(4, 4, generator=torch.Generator().manual_seed(5))
    a, b = tgt.make_cache(8), tgt.make_cache(8)
    want = tgt.sampled_round(3, draft, a, uniforms=u.t().reshape(-1).clone(), top_k=50)
    got = tgt.sampled_round(3, draft, b, uniforms=u.t(), top_k=50)
    assert got[:2] == want[:2] and a[0].offset == b[0].offset == got[0] + 1
