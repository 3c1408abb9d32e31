"""GPU: ops.rope against the rotation in 64 bits.

The angle is exact to 1e-9 rad and its fp32 form, in half turns below 1, to 2^-25 of them: pi 2^-25 rad. sin
and cos of it within two units (2^-22): each of the two products is off by at most 2^-21.5 |x| and the fp32
sum by 2^-23 (|x1| + |x2|) more: (|x1| + |x2|) 2^-21 together, then half a step of the type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(x, y, pos, freqs, inter, scale=1.0):
    """x, y [B, H, L, D]; pos [B, L] int64."""
    v = x.double().cpu().numpy()
    got = y.double().cpu().numpy()
    half = freqs.numel()
    first = np.arange(half) * (2 if inter else 1)
    second = first + (1 if inter else half)
    turn = scale * np.exp(1j * (pos.cpu().numpy().astype(np.float64)[:, None, :, None] * freqs.cpu().numpy()))
    z = (v[..., first] + 1j * v[..., second]) * turn
    want = v.copy()
    want[..., first], want[..., second] = z.real, z.imag
    tol = np.zeros_like(v)
    size = (np.abs(v[..., first]) + np.abs(v[..., second])) * scale * 2.0 ** -21
    tol[..., first] = tol[..., second] = size
    fi = torch.finfo(y.dtype)
    tol[..., :2 * half] += (np.abs(want) + tol)[..., :2 * half] * fi.eps / 2 + fi.smallest_normal * fi.eps
    assert y.dtype == x.dtype and got.shape == v.shape
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) - tol).max())


def make(g, B, H, L, D, dtype, dev):
    return torch.randn(B, L, H * D, generator=g).to(DT[dtype]).to(dev).view(B, L, H, D).transpose(1, 2)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,L,hq,hk,D,dims", [(1, 1, 32, 8, 128, 128), (3, 13, 6, 2, 256, 64), (1, 1100, 5, 1, 64, 64),
                                              (2, 3, 3, 3, 80, 40), (2, 5, 2, 1, 80, 20), (1, 7, 1, 1, 2, 2),
                                              (1, 2, 1, 1, 1024, 256), (2, 9, 4, 0, 96, 96), (1, 3, 2, 1, 65, 6),
                                              (1030, 1, 2, 1, 128, 128)])
def test_rope(dev, B, L, hq, hk, D, dims, dtype, inter):
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(B * 100 + L + D)
    freqs, _ = rope.frequencies(dims, 1e6, device=dev)
    q = make(g, B, hq, L, D, dtype, dev)
    k = make(g, B, hk, L, D, dtype, dev) if hk else None
    for pos in (7, 1 << 20, torch.randint(0, 1 << 20, (B, L), generator=g).to(dev),
                torch.randint(0, 1 << 20, (L,), generator=g).to(torch.int32).to(dev),
                torch.randint(0, 1 << 20, (B, 1), generator=g).to(dev), torch.randint(-9, 9, (L, B), generator=g).to(dev).t()):
        at = pos.expand(B, L) if isinstance(pos, torch.Tensor) else torch.arange(pos, pos + L).expand(B, L)
        scale = 1.0 if isinstance(pos, int) else 1.25
        yq, yk = ops.rope(q, k, freqs, pos, interleaved=inter, scale=scale)
        check(q, yq, at, freqs, inter, scale)
        assert (yk is None) == (k is None)
        if k is not None:
            check(k, yk, at, freqs, inter, scale)


@pytest.mark.parametrize("inter", [False, True])
def test_in_place_views_and_cache_rows(dev, inter):
    """Slices of one projection rotated where they are; keys into a cache's rows, the rows beside them kept; single
    values where a view starts off the 16 bytes; a transposed head dim."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(1)
    freqs, scale = rope.frequencies(64, 1e4, dict(type="yarn", factor=4.0, original_max_position_embeddings=2048), device=dev)
    B, L, hq, hk, D = 2, 6, 4, 2, 128
    pos = torch.randint(0, 9000, (B, L), generator=g).to(dev)
    for shift in (0, 1):
        buf = torch.randn(B, L, (hq + 2 * hk) * D + 8, generator=g).to(torch.bfloat16).to(dev)
        heads = lambda lo, h: buf[:, :, lo + shift:lo + shift + h * D].view(B, L, h, D).transpose(1, 2)
        q, k = heads(0, hq), heads(hq * D, hk)
        q0, k0, before = q.clone(), k.clone(), buf.clone()
        cache = torch.full((B, hk, 20, D), 9.0, dtype=torch.bfloat16, device=dev)
        rows = cache[:, :, 5:5 + L]
        yq, yk = ops.rope(q, k, freqs, pos, interleaved=inter, scale=scale, q_out=q, k_out=rows)
        assert yq is q and yk is rows
        check(q0, q, pos, freqs, inter, scale)
        check(k0, rows, pos, freqs, inter, scale)
        assert (cache[:, :, :5] == 9).all() and (cache[:, :, 5 + L:] == 9).all()
        heads(0, hq).copy_(q0)
        assert torch.equal(buf, before)
    t = torch.randn(B, D, L, hq, generator=g).to(torch.float16).to(dev).permute(0, 3, 2, 1)
    check(t, ops.rope(t, None, freqs, pos, interleaved=inter)[0], pos, freqs, inter)


def test_refusals(dev):
    from dspark_rocm import ops, rope

    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16, device=dev)
    f = rope.frequencies(64, 1e4, device=dev)[0]
    buf = torch.zeros(2, 4, 4, 64, dtype=torch.bfloat16, device=dev)
    for args, kw in (((q[0], k, f, 0), {}), ((q, k[:1], f, 0), {}), ((q, k[:, :, :2], f, 0), {}), ((q, k, f.float(), 0), {}),
                     ((q, k, torch.zeros(33, dtype=torch.float64, device=dev), 0), {}), ((q, k, f[:0], 0), {}), ((q, k, f.cpu(), 0), {}),
                     ((q, k, f, torch.zeros(2, 2, dtype=torch.int64, device=dev)), {}), ((q, k, f, torch.zeros(3, device=dev)), {}),
                     ((q, k, f, torch.zeros(3, dtype=torch.int64)), {}), ((q, k, f, 0), dict(q_out=q[:1])),
                     ((q, k, f, 0), dict(q_out=q.float())), ((q, None, f, 0), dict(k_out=k)),
                     ((buf[:, :, :3], None, f, 0), dict(q_out=buf[:, :, 1:])),
                     ((q, k, f, 0), dict(k_out=k[:, :, :1].expand(2, 1, 3, 64))),
                     ((q.float().requires_grad_(), None, f, 0), {})):
        with pytest.raises(ValueError):
            ops.rope(*args, **kw)
    for args in ((q.double(), None, f, 0), (q, k.half(), f, 0)):
        with pytest.raises(TypeError):
            ops.rope(*args)
    assert ops.rope(q[:0], k[:0], f, 0)[0].shape == (0, 4, 3, 64)
    assert ops.rope(q[:, :0], k[:, :0], f, 0)[1].shape == (2, 0, 3, 64)


def test_no_query_heads(dev):
    """Keys alone go as q."""
    from dspark_rocm import ops, rope

    k = make(torch.Generator().manual_seed(0), 1, 3, 4, 64, "bf16", dev)
    f = rope.frequencies(64, 1e4, device=dev)[0]
    with pytest.raises(Exception):
        ops.rope(k[:, :0], k, f, 0)
    check(k, ops.rope(k, None, f, 3)[0], torch.arange(3, 7)[None], f, False)


def test_stream_and_graph(dev):
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(2)
    q, k = make(g, 2, 8, 5, 128, "bf16", dev), make(g, 2, 2, 5, 128, "bf16", dev)
    f = rope.frequencies(128, 1e4, device=dev)[0]
    pos = torch.randint(0, 5000, (2, 5), generator=g).to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.rope(q, k, f, pos)
    s.synchronize()
    check(q, y[0], pos, f, False)
    check(k, y[1], pos, f, False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = ops.rope(q, k, f, pos)
    for _ in range(3):
        pos.copy_(torch.randint(0, 5000, (2, 5), generator=g))     # positions move on between replays
        graph.replay()
        want = ops.rope(q, k, f, pos)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(z, want))


@pytest.mark.parametrize("scale", [1.0, 1.25, 0.1 * np.log(4.0) + 1.0])
@pytest.mark.parametrize("inter", [False, True])
def test_small_values_of_a_turn(dev, inter, scale):
    """Unit vectors in fp32: their turn is the table itself, also where a cosine or sine is near zero. Each is within 4
    units of its own value (2^-21, the bound of sinpi and cospi), half a step for the rounding after the factor, and the
    angle: up to 2^13 radians, four roundings of 2^-53 and what an fp32 remainder of the half turns leaves (2^-50): under
    2^-37 together."""
    from dspark_rocm import ops, rope

    freqs, _ = rope.frequencies(128, 1e6, device=dev)
    L = 5000
    x = torch.zeros(1, 1, L, 128, device=dev)
    x[..., slice(0, 128, 2) if inter else slice(0, 64)] = 1.0
    y = ops.rope(x, None, freqs, 0, interleaved=inter, scale=scale)[0][0, 0].double().cpu().numpy()
    c, s = (y[:, ::2], y[:, 1::2]) if inter else (y[:, :64], y[:, 64:])
    a = np.arange(L)[:, None].astype(np.longdouble) * freqs.cpu().numpy().astype(np.longdouble)
    for got, want in ((c, np.cos(a) * scale), (s, np.sin(a) * scale)):
        assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -21 + 2.0 ** -24) + 2.0 ** -37).all()


def test_negated_views(dev):
    """The imaginary part of a conjugate, and one whose memory could be read as it lies: their values are rotated."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(6)
    f = rope.frequencies(64, 1e4, device=dev)[0]
    z = torch.randn(1, 2, 3, 64, dtype=torch.complex64, generator=g).to(dev)
    for q in (z.conj().imag, torch._neg_view(z.imag.clone())):
        assert q.is_neg()
        for y in ops.rope(q, q, f, 5):
            check(-z.imag, y, torch.arange(5, 8)[None], f, False)
