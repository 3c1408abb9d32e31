"""CPU: what the paged-cache operators refuse, copy and hand to their launches. The launches are left out: what is
refused is refused on the host before them."""

from __future__ import annotations

import struct

import pytest
import torch
from torch.autograd import forward_ad

from dspark_rocm import ops

BF = torch.bfloat16


@pytest.fixture
def host(monkeypatch):
    """The operators' host code on CPU tensors; the calls that would have been made."""
    calls = []
    monkeypatch.setattr(ops, "_one_device", lambda what, first, *ts: first.device)
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, args: calls.append((name, struct.unpack(f"={len(args) // 8}q", args))))
    return calls


def ids(*x):
    return torch.tensor(x, dtype=torch.int32)


def pages(codes=False, pool=5, Hk=2, P=16, D=64, dtype=BF):
    if codes:
        return torch.zeros(pool, Hk, P, D).to(torch.float8_e4m3fn), torch.zeros(pool, Hk, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return torch.zeros(pool, Hk, P, D, dtype=dtype)


def case(codes=False, **kw):
    row = lambda h: torch.zeros(3, h, 64, dtype=BF)
    d = dict(k=row(2), v=row(2), k_pages=pages(codes), v_pages=pages(codes), table=ids(0, 1, 2, 3).view(2, 2), starts=ids(0, 1, 3),
             lens=ids(4, 9), q=row(4), freqs=torch.zeros(32, dtype=torch.float64))
    d.update(kw)
    return d


def append(d):
    return ops.paged_append(**d)


def test_fields(host):
    for codes in (False, True):
        d = case(codes, positions=torch.arange(6)[::2], interleaved=True)
        y = append(d)
        name, f = host.pop()
        parts = lambda p: (p[0].data_ptr(), 2048, 1024, 64, p[1].data_ptr(), 2, 1) if codes else (p.data_ptr(), 2048, 1024, 64, 0, 0, 0)
        one = struct.unpack("=q", struct.pack("=d", 1.0))[0]
        assert name == "dspark_paged_append" and f == (
            0, codes, 4, 2, 64, 16, 5, 64, 1, d["freqs"].data_ptr(), one, d["positions"].data_ptr(), 1, 2, d["q"].data_ptr(), 256, 64,
            y.data_ptr(), 256, 64, 1, d["k"].data_ptr(), 128, 64, d["v"].data_ptr(), 128, 64, *parts(d["k_pages"]), *parts(d["v_pages"]),
            d["table"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), 2, 2, 2, 3)
        k, v = ops.paged_read(d["k_pages"], d["v_pages"], ids(1, 2, 2), dtype=BF)
        name, f = host.pop()
        assert name == "dspark_paged_read" and f[:6] == (0, codes, 2, 64, 16, 5) and f[7] == 3 and f[-2:] == (k.data_ptr(), v.data_ptr())


def test_refused_appends(host):
    z = torch.zeros
    p8 = pages(True)
    bad = [dict(k=z(3, 2, 64)), dict(k=z(3, 3, 64, dtype=BF)), dict(k=z(2, 2, 64, dtype=BF)), dict(k=z(3, 2, 128, dtype=BF)),
           dict(v=z(3, 2, 64, dtype=torch.float16)), dict(q=z(3, 4, 64)), dict(q=z(2, 4, 64, dtype=BF)), dict(q=z(3, 256, dtype=BF)),
           dict(k_pages=pages(P=8)), dict(k_pages=pages(D=80)), dict(k_pages=pages(pool=4)), dict(k_pages=pages(dtype=torch.float16)),
           dict(k_pages=p8), dict(k_pages=(p8[0], p8[1].view(torch.uint8)), v_pages=pages(True)),
           dict(k_pages=(p8[0], p8[1][:4]), v_pages=pages(True)), dict(k_pages=pages().transpose(2, 3)),
           dict(k_pages=pages(pool=1).expand(5, 2, 16, 64)), dict(table=ids(0, 1)), dict(table=z(2, 2)), dict(starts=ids(0, 3)),
           dict(starts=z(3)), dict(lens=ids(4)), dict(lens=z(2)), dict(freqs=z(32)), dict(freqs=z(33, dtype=torch.float64)),
           dict(freqs=z(12, dtype=torch.float64)), dict(freqs=z(0, dtype=torch.float64)), dict(positions=ids(0, 1)),
           dict(positions=z(3)), dict(q=None, q_out=z(3, 4, 64, dtype=BF)), dict(q_out=z(3, 4, 64)), dict(q_out=z(2, 4, 64, dtype=BF)),
           dict(q_out=z(3, 4, 128, dtype=BF)[..., ::2]), dict(q_out=z(3, 1, 64, dtype=BF).expand(3, 4, 64)),
           dict(table=z(4097, 1, dtype=torch.int32), starts=z(4098, dtype=torch.int32), lens=z(4097, dtype=torch.int32))]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            append(case(**kw))
    d = case()
    for kw in (dict(v_pages=d["k_pages"]), dict(q=d["q"][:, :2], q_out=d["k"]), dict(q=d["q"][:, :2], q_out=d["k_pages"][0].view(2, 16, 64)[:, :3].transpose(0, 1))):
        with pytest.raises(ValueError, match="twice"):
            append({**d, **kw})
    buf = z(4, 4, 64, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        append(case(q=buf[:3], q_out=buf[1:]))
    assert not host


def test_sizes_of_nothing(host):
    d = case()
    none = dict(k=d["k"][:0], v=d["v"][:0], q=d["q"][:0])
    assert append({**d, **none}).shape == (0, 4, 64)
    y = append({**d, "table": d["table"][:0], "starts": ids(0), "lens": ids()})
    assert y.shape == (3, 4, 64) and not y.any()
    assert ops.paged_read(d["k_pages"], d["v_pages"], ids())[0].shape == (0, 2, 16, 64)
    assert not host
    assert append({**d, "q": None}) is None and len(host) == 1


def test_copies_where_addresses_need_them(host):
    wide = torch.zeros(3, 2, 65, dtype=BF)
    d = case(k=wide[..., 1:], table=torch.zeros(2, 4, dtype=torch.int64)[:, ::2], starts=torch.tensor([0, 1, 3]))
    append(d)
    f = host.pop()[1]
    assert f[21] != d["k"].data_ptr() and f[22:24] == (128, 64)
    assert f[-4] == 2 and f[-7] % 4 == 0
    with pytest.raises(ValueError):
        append(case(q_out=torch.zeros(3, 4, 65, dtype=BF)[..., 1:]))


@pytest.mark.parametrize("name", ["k", "v", "q", "freqs", "k_pages", "v_pages", "q_out"])
def test_gradients_and_tangents_are_not_dropped(host, name):
    d = case(q_out=torch.zeros(3, 4, 64, dtype=BF))
    append(d)
    d[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        append(d)
    with torch.no_grad():
        append(d)
    d[name].requires_grad_(False)
    with forward_ad.dual_level():
        d[name] = forward_ad.make_dual(d[name], torch.ones_like(d[name]))
        with pytest.raises(ValueError, match="tangent"):
            append(d)
    assert len(host) == 2


@pytest.mark.parametrize("name", ["k", "v", "q", "freqs", "k_pages", "v_pages", "q_out"])
def test_negated_views(host, name):
    d = case(q_out=torch.zeros(3, 4, 64, dtype=BF))
    plain = d[name]
    d[name] = torch._neg_view(plain)
    if name in ("k_pages", "v_pages", "q_out"):
        with pytest.raises(ValueError, match="negates"):
            append(d)
    else:
        append(d)
        assert plain.data_ptr() not in host.pop()[1]


# ---------------------------------------------------------------------------- attention


def attend(d, **kw):
    d = {n: t for n, t in d.items() if n not in ("k", "v", "freqs")}
    return ops.paged_attention(**{"scale": 0.5, **d, **kw})


def test_attention_fields(host):
    for codes in (False, True):
        d = case(codes)
        y = attend(d, max_rows=2, max_len=17, causal=False)
        name, f = host.pop()
        half = struct.unpack("=q", struct.pack("=d", 0.5))[0]
        assert name == "dspark_paged_attention"
        assert f[:17] == (0, codes, 4, 2, 64, 16, 5, 0, 1, 2, half, d["q"].data_ptr(), 256, 64, y.data_ptr(), 256, 64)
        assert f[-9:-2] == (d["table"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), 2, 2, 2, 3) and f[-1] >= 256
        attend(d, max_len=16, max_rows=7)
        f = host.pop()[1]
        assert f[9] == 3 and f[-4] == 1
        out = torch.zeros(3, 8, 64, dtype=BF)[:, 4:]
        ws = torch.zeros(ops.paged_attention_workspace_bytes(2, 4, 2, 64, 3, 3, 32), dtype=torch.uint8)
        assert attend(d, out=out, workspace=ws) is out
        f = host.pop()[1]
        assert f[8] == 0 and f[14:17] == (out.data_ptr(), 512, 64) and f[-2:] == (ws.data_ptr(), ws.numel())


def test_refused_attention(host):
    z = torch.zeros
    d = case()
    bad = [dict(q=z(3, 4, 64)), dict(q=z(3, 3, 64, dtype=BF)), dict(q=z(3, 4, 128, dtype=BF)), dict(q=z(12, 64, dtype=BF)), dict(scale=0.0),
           dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(max_rows=0), dict(max_len=-20), dict(v_pages=pages(pool=4)),
           dict(v_pages=pages(True)), dict(k_pages=pages(P=8), v_pages=pages(P=8)), dict(out=z(3, 4, 64)), dict(out=z(2, 4, 64, dtype=BF)),
           dict(out=z(3, 1, 64, dtype=BF).expand(3, 4, 64)), dict(out=z(3, 4, 65, dtype=BF)[..., 1:]), dict(out=d["q"]),
           dict(out=torch._neg_view(z(3, 4, 64, dtype=BF))), dict(workspace=z(8, dtype=torch.uint8)), dict(workspace=z(10 ** 7, dtype=torch.uint8)[1:]),
           dict(starts=ids(0, 3)), dict(lens=ids(1)), dict(table=z(2, 2)),
           dict(table=z(1, 1, dtype=torch.int32).expand(2, 1 << 27))]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            attend(d, **kw)
    assert not host


def test_attention_of_nothing(host):
    d = case()
    assert attend({**d, "q": d["q"][:0]}).shape == (0, 4, 64)
    assert not attend({**d, "table": d["table"][:0], "starts": ids(0), "lens": ids()}).any()
    assert not attend({**d, "table": d["table"][:, :0]}).any() and not attend(d, max_len=0).any()
    out = torch.ones(3, 4, 64, dtype=BF)
    assert attend(d, max_len=0, out=out) is out and (out == 1).all()
    assert not host


@pytest.mark.parametrize("name", ["q", "k_pages", "v_pages", "out"])
def test_attention_derivatives_and_negated_views(host, name):
    d = case(out=torch.zeros(3, 4, 64, dtype=BF))
    d[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        attend(d)
    with torch.no_grad():
        attend(d)
    d[name].requires_grad_(False)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            attend({**d, name: forward_ad.make_dual(d[name], torch.ones_like(d[name]))})
    plain, d[name] = d[name], torch._neg_view(d[name])
    if name == "q":
        attend(d)
        assert plain.data_ptr() not in host.pop()[1]
    else:
        with pytest.raises(ValueError, match="negates"):
            attend(d)


def test_plans_fit_their_workspace():
    """Every plan's workspace is what the entry point asks for; too much for one call is refused."""
    f = ops.paged_attention_workspace_bytes
    assert f(1, 32, 8, 128, 1, 1, 512) == 256                      # whole rows: nothing to join
    assert f(1, 32, 8, 128, 1, 1, 32768) == 512 * 2 * 16 * 130 * 4
    assert f(32, 32, 8, 128, 32, 1, 640) == 512 * 2 * 16 * 130 * 4
    assert f(1, 8, 8, 64, 1, 1, 640) == 40 * 2 * 16 * 66 * 4       # no more workgroups than units
    assert f(1, 32, 8, 100, 1, 1, 512) == 0 and f(4097, 8, 8, 64, 1, 1, 64) == 0 and f(1, 9, 8, 64, 1, 1, 64) == 0
    assert f(4096, 64, 64, 64, 1 << 21, 1, 1 << 30) == 0


# ---------------------------------------------------------------------------- scores


def test_refused_scores(host):
    z = torch.zeros
    for x, t, kw in ((z(3, 9, dtype=torch.float64), ids(0, 1, 2), {}), (z(3, 9, dtype=torch.int32), ids(0, 1, 2), {}),
                     (z(3, 9), ids(0, 1), {}), (z(3, 9), z(3), {}), (z(3, 9), ids(0, 1, 2).view(3, 1), {}), (z(3, 0), ids(0, 1, 2), {}),
                     (z(3, 9), ids(0, 1, 2), dict(top=10)), (z(3, 99), ids(0, 1, 2), dict(top=65)), (z(3, 9), ids(0, 1, 2), dict(top=-1)),
                     (z(3, 9), ids(0, 1, 2), dict(temperature=0.0)), (z(3, 9), ids(0, 1, 2), dict(temperature=float("nan"))),
                     (z(3, 9), ids(0, 1, 2), dict(workspace=z(8, dtype=torch.uint8))), (z(()), ids(0), {}),
                     (z(3, 9).requires_grad_(), ids(0, 1, 2), {}), (z(1, 1).expand(3, 1 << 29), ids(0, 1, 2), {})):
        with pytest.raises((ValueError, TypeError)):
            ops.token_logprobs(x, t, **kw)
    assert not host


def test_score_fields(host):
    x = torch.zeros(2, 3, 10, dtype=torch.float16)[..., :9]
    g, h, i, b = ops.token_logprobs(x[:, :2], torch.zeros(2, 2, dtype=torch.int64), top=4, temperature=0.5)
    name, f = host.pop()
    assert name == "dspark_token_logprobs" and f[0] == 1 and f[3:5] == (4, 9) and f[6:8] == (1, 4)
    assert f[9:13] == (g.data_ptr(), h.data_ptr(), i.data_ptr(), b.data_ptr()) and i.shape == b.shape == (2, 2, 4)
    y = torch.zeros(5, 9)
    ops.token_logprobs(y, ids(0, 1, 2, 3, 4))
    f = host.pop()[1]
    assert f[1:5] == (y.data_ptr(), 9, 5, 9) and f[6] == 0
    ops.token_logprobs(torch._neg_view(y), ids(0, 1, 2, 3, 4))
    assert host.pop()[1][1] != y.data_ptr()
    assert ops.token_logprobs(y[:0], ids(), top=3)[2].shape == (0, 3) and not host
    one = ops.token_logprobs(y[0], torch.tensor(3, dtype=torch.int32), top=2)
    assert one[0].shape == () and one[3].shape == (2,) and len(host) == 1
