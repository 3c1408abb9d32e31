"""GPU: quantize_kv and dequantize_kv against the quantizer's rule in fp64 (each of its steps rounded to fp32,
which rounds as fp32 operations do: 53 bits are over 2 * 24 + 2), and against quant.quantize_rows: equal bits.
The quotient by 2^bits - 1 is a product with its rounded reciprocal, as torch's ops form it on this GPU."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def rule(x, bits, cdt):
    """(fields, scales, biases) of x [..., D], on the CPU."""
    r32 = lambda a: a.to(torch.float32).double()
    v = x.detach().cpu().double().reshape(*x.shape[:-1], -1, 64)
    lo, hi, levels = v.amin(-1), v.amax(-1), 2 ** bits - 1
    s, b = (r32(hi - lo) * r32(torch.tensor(1.0).double() / levels)).to(torch.float32).to(cdt), lo.to(torch.float32).to(cdt)
    div = torch.where(s == 0, 1.0, s.double())
    f = torch.round(r32(r32(v - b.double()[..., None]) / div[..., None])).clamp(0, levels)
    return torch.nan_to_num(f, 0.0).to(torch.int64).flatten(-2), s, b


def fields(w, bits):
    f = torch.stack([(w.cpu().to(torch.int64) & 0xFFFFFFFF) >> (bits * j) & (2 ** bits - 1) for j in range(32 // bits)], -1)
    return f.flatten(-2)


def cache(B, H, cap, D, bits, cdt, dev, odd=0):
    """A (words, scales, biases) triple of sentinels; odd: the words start 4 bytes off the 16."""
    n = D * bits // 32
    w = torch.full((B * H * cap * n + odd,), 0x5A5A5A5A, dtype=torch.int32, device=dev)[odd:].view(B, H, cap, n)
    s = torch.full((B, H, cap, D // 64), 7.0, dtype=cdt, device=dev)
    return w, s, s.clone()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.cpu().float(), 77.0), torch.nan_to_num(b.cpu().float(), 77.0))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("src,cdt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("B,H,T,D,at", [(1, 8, 1, 128, 0), (2, 3, 5, 64, 7), (1, 4, 300, 256, 100), (3, 1, 17, 192, 1)])
def test_write_and_read(dev, B, H, T, D, at, src, cdt, bits):
    from dspark_rocm import ops, quant

    g = torch.Generator().manual_seed(T + D)
    cap = at + T + 3
    x = [torch.randn(B, T, H * D, generator=g).to(DT[src]).to(dev).view(B, T, H, D).transpose(1, 2) for _ in range(2)]
    x[0][:, :, 0, :64] = 1.5                                            # a group of one value: scale 0
    for odd in (0, 1):
        trips = [cache(B, H, cap, D, bits, DT[cdt], dev, odd) for _ in range(2)]
        before = [[t.clone() for t in trip] for trip in trips]
        ops.quantize_kv(*x, *[tuple(t[:, :, at:at + T] for t in trip) for trip in trips], bits=bits)
        for trip, old, rows in zip(trips, before, x):
            f, s, b = rule(rows, bits, DT[cdt])
            assert torch.equal(fields(trip[0][:, :, at:at + T], bits), f)
            assert torch.equal(trip[1][:, :, at:at + T].cpu(), s) and torch.equal(trip[2][:, :, at:at + T].cpu(), b)
            for t, o, q in zip(trip, old, quant.quantize_rows(rows, bits, dtype=DT[cdt])):
                assert torch.equal(t[:, :, at:at + T], q)
                assert torch.equal(t[:, :, :at], o[:, :, :at]) and torch.equal(t[:, :, at + T:], o[:, :, at + T:])
        for dt in (torch.float32, DT[cdt], torch.float16):
            got = ops.dequantize_kv(*[tuple(t[:, :, :at + T] for t in trip) for trip in trips], bits=bits, dtype=dt)
            for trip, y in zip(trips, got):
                q = fields(trip[0][:, :, :at + T], bits).double().unflatten(-1, (-1, 64))
                s, b = (t[:, :, :at + T].cpu().double()[..., None] for t in trip[1:])
                want = ((q * s).to(torch.float32).double() + b).to(torch.float32).flatten(-2).to(dt)
                assert y.dtype == dt and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_values_that_are_not_finite(dev, dtype, bits):
    """NaN, infinities and the type's ends: what quantize_rows and the read back make of them."""
    from dspark_rocm import ops, quant

    x = torch.randn(1, 1, 8, 64, generator=torch.Generator().manual_seed(0)).to(DT[dtype]).to(dev)
    fi = torch.finfo(DT[dtype])
    for r, v in enumerate((float("nan"), float("inf"), float("-inf"), fi.max, fi.min, fi.tiny)):
        x[0, 0, r, 11 * r] = v
    x[0, 0, 6] = float("inf")
    x[0, 0, 7, ::2], x[0, 0, 7, 1::2] = fi.max, fi.min
    trips = [cache(1, 1, 8, 64, bits, torch.bfloat16, dev) for _ in range(2)]
    ops.quantize_kv(x, x, *trips, bits=bits)
    w, s, b = quant.quantize_rows(x, bits)
    for trip in trips:
        assert torch.equal(trip[0], w) and same(trip[1], s) and same(trip[2], b)
    y = ops.dequantize_kv(*trips, bits=bits)
    f = fields(w, bits).float().unflatten(-1, (-1, 64))
    want = (f * s.cpu().float()[..., None] + b.cpu().float()[..., None]).flatten(-2)
    assert same(y[0], want) and same(y[1], want)


def test_offsets_past_32_bits(dev):
    """Heads more than 2^31 elements apart."""
    from dspark_rocm import ops

    far = (1 << 31) + 512
    buf = torch.empty(far + 4096, dtype=torch.int32, device=dev)
    w = buf.as_strided((1, 2, 16, 32), (0, far, 32, 1))
    s = torch.zeros(1, 2, 16, 2, dtype=torch.bfloat16, device=dev)
    rows = torch.empty(far + 4096, dtype=torch.bfloat16, device=dev).as_strided((1, 2, 16, 128), (0, far, 128, 1))
    rows.copy_(torch.randn(1, 2, 16, 128, generator=torch.Generator().manual_seed(0)))
    v = cache(1, 2, 16, 128, 8, torch.bfloat16, dev)
    ops.quantize_kv(rows, rows, (w, s, s.clone()), v, bits=8)
    assert torch.equal(w, v[0])
    out = torch.empty(far + 4096, dtype=torch.bfloat16, device=dev).as_strided((1, 2, 16, 128), (0, far, 128, 1))
    got = ops.dequantize_kv((w, v[1], v[2]), v, bits=8, dtype=torch.bfloat16, out=(out, torch.empty_like(out)))
    assert torch.equal(got[0], got[1])
    from dspark_rocm import rope

    f = rope.frequencies(128, 1e4, device=dev)[0]
    assert torch.equal(ops.rope(rows, None, f, 5, q_out=out)[0], ops.rope(rows.contiguous(), None, f, 5)[0])


def test_refusals(dev):
    from dspark_rocm import ops

    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device=dev)
    w, s, b = cache(1, 2, 3, 64, 8, torch.bfloat16, dev)
    t = (w, s, b)
    for args, kw in (((x, x[:, :1], t, t), {}), ((x, x, (w[:, :, :2], s, b), t), {}), ((x, x, t, (w, s[:, :, :2], b)), {}),
                     ((x, x, t, t), dict(bits=4)), ((x, x, t, t), dict(bits=3)), ((x, x, t, t), dict(group_size=32)),
                     ((x, x, (w, s, b[:, :, :, :1].expand_as(b).transpose(1, 2).contiguous().transpose(1, 2)), t), {}),
                     ((x.cpu(), x, t, t), {}), ((x.float().requires_grad_(), x.float(), t, t), {}),
                     ((x, x, (w[:, :, :1].expand_as(w), s, b), t), {})):
        with pytest.raises(ValueError):
            ops.quantize_kv(*args, **{**dict(bits=8), **kw})
    for args in ((x.double(), x.double(), t, t), (x, x.half(), t, t), (x, x, (w, s.float(), b.float()), t), (x, x, (w.long(), s, b), t),
                 (x, x, t, (w, s.half(), b.half()))):
        with pytest.raises(TypeError):
            ops.quantize_kv(*args, bits=8)
    for bad in (dict(out=(x, x)), dict(out=(x.float(), x.float()[:, :1])), dict(bits=4),
                dict(out=(x.float(), torch.zeros(1, 1, 3, 64, device=dev).expand(1, 2, 3, 64)))):
        with pytest.raises(ValueError):
            ops.dequantize_kv(t, t, **{**dict(bits=8), **bad})
    with pytest.raises(TypeError):
        ops.dequantize_kv(t, t, bits=8, dtype=torch.float64)
    empty = tuple(a[:, :, :0] for a in t)
    ops.quantize_kv(x[:, :, :0], x[:, :, :0], empty, empty, bits=8)
    assert ops.dequantize_kv(empty, empty, bits=8)[0].shape == (1, 2, 0, 64)


@pytest.mark.parametrize("bits", [4, 8])
def test_the_cache_and_the_stock_attention_take_them(dev, bits, monkeypatch):
    """The same bits as the torch ops they stand in for; calls autograd follows keep those."""
    from dspark_rocm import fast, ops
    from dspark_rocm.kv_cache import QuantizedKVCache

    g = torch.Generator().manual_seed(bits)
    rows = [torch.randn(2, 2, 300, 64, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)]
    q = torch.randn(2, 4, 5, 64, generator=g).to(torch.bfloat16).to(dev)
    calls = []
    for name in ("quantize_kv", "dequantize_kv"):
        real = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, _r=real, _n=name, **k: calls.append(_n) or _r(*a, **k))

    def use(q, *rows):
        c = QuantizedKVCache(2, 2, 64, bits=bits, device=dev)
        c.update_and_fetch(*(r[:, :, :1] for r in rows))
        keys, values = c.update_and_fetch(*(r[:, :, 1:] for r in rows))         # grows
        return fast.quantized_scaled_dot_product_attention(q, keys, values, scale=0.125, mask="causal", bits=bits), *keys, *values

    got = use(q, *rows)
    assert calls == ["quantize_kv", "quantize_kv", "dequantize_kv"]
    calls.clear()
    monkeypatch.setattr(ops, "eager_inference", lambda *ts: False)
    want = use(q, *rows)
    assert not calls and all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.undo()
    q.requires_grad_()
    out = use(q, *rows)[0]
    out.float().sum().backward()
    assert torch.equal(out, want[0]) and bool(torch.isfinite(q.grad).all())


def test_stream_and_graph(dev):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(2)
    x = [torch.randn(1, 2, 6, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)]
    trips = [cache(1, 2, 6, 128, 8, torch.bfloat16, dev) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.quantize_kv(*x, *trips, bits=8)
        y = ops.dequantize_kv(*trips, bits=8)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.quantize_kv(*x, *trips, bits=8)
        z = ops.dequantize_kv(*trips, bits=8)
    assert all(float((a - b.float()).abs().max()) < 0.1 for a, b in zip(y, x))
    for _ in range(3):
        for t in x:
            t.copy_(torch.randn(1, 2, 6, 128, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in z]
        ops.quantize_kv(*x, *trips, bits=8)
        assert all(torch.equal(a, b) for a, b in zip(kept, ops.dequantize_kv(*trips, bits=8)))


def test_rows_given_twice(dev):
    """Rows that two workgroups would write, or one write while another reads: refused."""
    from dspark_rocm import ops, rope

    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device=dev)
    t, u = (cache(1, 2, 3, 64, 8, torch.bfloat16, dev) for _ in range(2))
    for k_rows, v_rows in ((t, t), ((t[0], t[1], t[1]), u), (t, (u[0], t[1], u[2]))):
        with pytest.raises(ValueError, match="twice"):
            ops.quantize_kv(x, x, k_rows, v_rows, bits=8)
    out = torch.empty_like(x, dtype=torch.float32)
    with pytest.raises(ValueError, match="twice"):
        ops.dequantize_kv(t, u, bits=8, out=(out, out))
    f, y = rope.frequencies(64, 1e4, device=dev)[0], torch.zeros_like(x)
    for args, kw in (((x, y), dict(q_out=x, k_out=x)), ((x, x), dict(q_out=x)), ((x, y), dict(k_out=x)), ((x, y), dict(q_out=y))):
        with pytest.raises(ValueError):
            ops.rope(*args, f, 0, **kw)
    with pytest.raises(ValueError, match="backward"):
        ops.rope(x, None, f.clone().requires_grad_(), 0)
    ops.rope(x, y, f, 0, q_out=x, k_out=y)


def test_heads_past_the_kernel(dev):
    """Heads wider than the kernels take: the cache and its read back go by torch ops, as they did."""
    from dspark_rocm import fast
    from dspark_rocm.kv_cache import QuantizedKVCache
    from dspark_rocm.quant import quantize_rows

    D = 4096 + 64
    x = torch.randn(1, 1, 2, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    c = QuantizedKVCache(1, 1, D, bits=8, device=dev)
    keys, values = c.update_and_fetch(x, x)
    for got, want in zip(keys, quantize_rows(x, 8, 64, torch.bfloat16)):
        assert torch.equal(got, want)
    assert not fast.read_back_kernel(x, keys, values, 8, 64)


def test_a_cache_that_records(dev):
    """Scales and biases with gradients: neither written nor read back without them."""
    from dspark_rocm import ops

    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device=dev)
    t, u = (cache(1, 2, 3, 64, 8, torch.bfloat16, dev) for _ in range(2))
    for i in (1, 2):
        grad = tuple(a.clone().requires_grad_() if j == i else a for j, a in enumerate(t))
        for call in (lambda: ops.quantize_kv(x, x, grad, u, bits=8), lambda: ops.quantize_kv(x, x, u, grad, bits=8),
                     lambda: ops.dequantize_kv(grad, u, bits=8), lambda: ops.dequantize_kv(u, grad, bits=8)):
            with pytest.raises(ValueError, match="backward"):
                call()
        with torch.no_grad():
            assert torch.equal(ops.dequantize_kv(grad, u, bits=8)[0], ops.dequantize_kv(t, u, bits=8)[0])


def test_tangents(dev):
    """Duals are refused by the operators; the cache and the stock attention keep the torch ops for them."""
    from torch.autograd import forward_ad

    from dspark_rocm import fast, ops
    from dspark_rocm.kv_cache import QuantizedKVCache

    g = torch.Generator().manual_seed(0)
    rows = [torch.randn(1, 2, 30, 64, generator=g).to(dev) for _ in range(2)]
    q = torch.randn(1, 2, 3, 64, generator=g).to(dev)
    t, u = (cache(1, 2, 30, 64, 8, torch.bfloat16, dev) for _ in range(2))
    c = QuantizedKVCache(1, 2, 64, bits=8, device=dev)
    keys, values = c.update_and_fetch(*rows)
    attend = lambda q: fast.quantized_scaled_dot_product_attention(q, keys, values, scale=0.125, bits=8)
    want = attend(q)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(rows[0], torch.ones_like(rows[0]))
        with pytest.raises(ValueError, match="tangent"):
            ops.quantize_kv(dual, rows[1], t, u, bits=8)
        out = forward_ad.unpack_dual(attend(forward_ad.make_dual(q, torch.ones_like(q))))
        assert torch.equal(out.primal, want) and bool(out.tangent.abs().sum() > 0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("cdt", ["f16", "bf16"])
def test_scales_round_twice(dev, bits, cdt):
    """Ranges whose product with the reciprocal lies beside the middle of two scales, so close that it is there in fp32:
    the scale is the even one, as two roundings give it, on whichever side of the middle the product lies."""
    from dspark_rocm import ops, quant

    dt = DT[cdt]
    levels, ulp = 2 ** bits - 1, torch.finfo(dt).eps
    recip = torch.tensor(1.0 / levels, dtype=torch.float32).double()
    mid = 1.0 + ulp * (torch.arange(1 / ulp if cdt == "f16" else 128).double() + 0.5)
    d = torch.cat([(mid * levels).to(torch.float32).view(torch.int32) + i for i in (-1, 0, 1)]).view(torch.float32)
    exact, near = d.double() * recip, (d.double() * recip).to(torch.float32)
    m3 = mid.repeat(3)
    once = torch.where(exact > m3, m3 + ulp / 2, m3 - ulp / 2)
    twice = near.to(dt).double()
    d = d[(near.double() == m3) & (exact != m3) & (once != twice)]
    assert len(d) > 10
    x = torch.zeros(1, 1, len(d), 64)
    x[0, 0, :, 5] = d
    x = x.to(dev)
    trips = [cache(1, 1, len(d), 64, bits, dt, dev) for _ in range(2)]
    ops.quantize_kv(x, x, *trips, bits=bits)
    f, s, b = rule(x, bits, dt)
    for trip, q in zip(zip(*trips), quant.quantize_rows(x, bits, dtype=dt)):
        assert torch.equal(trip[0], trip[1]) and torch.equal(trip[0], q)
    assert torch.equal(trips[0][1].cpu(), s) and torch.equal(fields(trips[0][0], bits), f)
