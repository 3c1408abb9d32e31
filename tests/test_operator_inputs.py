"""CPU: tensors whose values are not what lies at their address, or that autograd follows, at the operators without a
backward pass. The launches are left out: what is refused is refused on the host before them."""

from __future__ import annotations

import struct

import pytest
import torch

from dspark_rocm import ops


@pytest.fixture
def host(monkeypatch):
    """The operators' host code on CPU tensors; the calls that would have been made."""
    calls = []
    monkeypatch.setattr(ops, "_one_device", lambda what, first, *ts: first.device)
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, args: calls.append(name))
    return calls


def _triple(dtype=torch.bfloat16):
    return [torch.zeros(1, 2, 3, 16, dtype=torch.int32), torch.zeros(1, 2, 3, 1, dtype=dtype), torch.zeros(1, 2, 3, 1, dtype=dtype)]


def _probs(logits, out):
    ops.sampling_probs(logits, out=out)


def _verify(logits, draft_probs):
    ops.speculative_verify(logits, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3), draft_probs=draft_probs)


def _rope(q, k, freqs, q_out, k_out):
    ops.rope(q, k, freqs, 3, q_out=q_out, k_out=k_out)


def _quantize(keys, values, ks, kb, vs, vb):
    (kw, _, _), (vw, _, _) = _triple(), _triple()
    ops.quantize_kv(keys, values, (kw, ks, kb), (vw, vs, vb), bits=8)


def _dequantize(ks, kb, vs, vb, k_out, v_out):
    (kw, _, _), (vw, _, _) = _triple(), _triple()
    ops.dequantize_kv((kw, ks, kb), (vw, vs, vb), bits=8, out=(k_out, v_out))


def _inputs():
    """Each operator with the tensors whose gradients it would have."""
    head = lambda: torch.zeros(1, 2, 3, 64)
    scale = lambda: torch.zeros(1, 2, 3, 1, dtype=torch.bfloat16)
    return [(_probs, dict(logits=torch.zeros(2, 9, dtype=torch.bfloat16), out=torch.zeros(2, 9))),
            (_verify, dict(logits=torch.zeros(2, 3, 9, dtype=torch.float16), draft_probs=torch.zeros(2, 2, 9))),
            (_rope, dict(q=head(), k=head(), freqs=torch.zeros(32, dtype=torch.float64), q_out=head(), k_out=head())),
            (_quantize, dict(keys=head(), values=head(), ks=scale(), kb=scale(), vs=scale(), vb=scale())),
            (_dequantize, dict(ks=scale(), kb=scale(), vs=scale(), vb=scale(), k_out=head(), v_out=head()))]


EACH = [(i, name) for i, (_, kw) in enumerate(_inputs()) for name in kw]


@pytest.mark.parametrize("i,name", EACH)
def test_gradients_are_not_dropped(host, i, name):
    call, kw = _inputs()[i]
    call(**kw)
    assert len(host) == 1
    kw[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        call(**kw)
    assert len(host) == 1
    with torch.no_grad():
        call(**kw)
    assert len(host) == 2


@pytest.mark.parametrize("i,name", EACH)
def test_tangents_are_not_dropped(host, i, name):
    """Forward mode does not ask for requires_grad, nor for grad mode."""
    from torch.autograd import forward_ad

    call, kw = _inputs()[i]
    with forward_ad.dual_level():
        call(**kw)                      # a level alone is no tangent
        assert len(host) == 1
        plain = kw[name]
        kw[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(ValueError, match="tangent"):
            call(**kw)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            call(**kw)
        assert len(host) == 1
        kw[name] = forward_ad.unpack_dual(kw[name]).primal
        call(**kw)
        assert len(host) == 2


class _Round:
    """What Target.sampled_round asks of a target, on the CPU; counts the verify steps."""

    max_rows = 16

    def __init__(self):
        from types import SimpleNamespace

        self.engine = SimpleNamespace(ids=torch.zeros(16, dtype=torch.int64))
        self.model = SimpleNamespace(args=SimpleNamespace(vocab_size=9))
        self.steps = 0

    def verify(self, ids, cache, tap):
        self.steps += 1
        return torch.zeros(1, ids.numel(), 9, dtype=torch.bfloat16), None

    def rollback(self, cache, n):
        pass


def test_round_refuses_tangents_before_the_caches_take_rows(host):
    from dspark_rocm.model import Target
    from torch.autograd import forward_ad

    r = _Round()
    with forward_ad.dual_level():
        q = forward_ad.make_dual(torch.zeros(2, 9), torch.ones(2, 9))
        with pytest.raises(ValueError):
            Target.sampled_round(r, 3, [1, 2], [], draft_probs=q)
    assert not r.steps


@pytest.mark.parametrize("i,name", EACH)
def test_negated_views_are_not_read_as_stored(host, monkeypatch, i, name):
    """A view that negates when it is read (as the imaginary part of a conjugate is): its memory holds other values.
    Plain inputs are copied, caches and outputs refused."""
    fields = []
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, args: fields.append(struct.unpack(f"={len(args) // 8}q", args)))
    call, kw = _inputs()[i]
    call(**kw)
    assert kw[name].data_ptr() in fields[0]
    view = kw[name] = torch._neg_view(kw[name])
    if name in ("logits", "draft_probs", "q", "k", "freqs", "keys", "values"):
        call(**kw)
        assert len(fields) == 2 and view.data_ptr() not in fields[1]
    else:
        with pytest.raises(ValueError, match="resolve_neg"):
            call(**kw)
        assert len(fields) == 1


def test_negated_uniforms(host, monkeypatch):
    fields = []
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, args: fields.append(struct.unpack(f"={len(args) // 8}q", args)))
    u = torch.full((2, 3), -0.25)
    for v in (u, torch._neg_view(u)):
        ops.speculative_verify(torch.zeros(2, 3, 9, dtype=torch.float16), torch.zeros(2, 2, dtype=torch.int32), v)
    assert u.data_ptr() in fields[0] and u.data_ptr() not in fields[1]


def test_zero_tensors_have_no_address(host):
    """A given tensor without memory is not taken for one that was not given."""
    with pytest.raises(ValueError):
        _verify(torch.zeros(2, 3, 9, dtype=torch.float16), torch._efficientzerotensor((2, 2, 9)))
    assert not host


def test_round_takes_uniforms_of_any_strides(host, monkeypatch):
    """They are formed before the verify step: one that cannot be viewed as a row would raise behind it, with the rows
    in the caches."""
    from dspark_rocm.model import Target

    seen = []

    def accept(logits, draft, uniforms, **kw):
        seen.append(uniforms)
        return None, torch.tensor([[4] + [-1] * 15]), None

    monkeypatch.setattr(ops, "speculative_verify", accept)
    u, r = torch.rand(4, 4), _Round()
    assert Target.sampled_round(r, 3, [1] * 15, [], uniforms=u.t())[:2] == (0, [4])
    assert r.steps == 1 and torch.equal(seen[0], u.t().reshape(1, 16))


def _other_buffers(name, trip):
    w, s, b = trip
    if name == "fp32 scales":
        return w, s.float(), b.float()
    if name == "biases of other strides":
        return w, s, b.transpose(1, 2).contiguous().transpose(1, 2)
    if name == "words of another stride":
        return w.transpose(2, 3).contiguous().transpose(2, 3), s, b
    return w.view(torch.uint32), s, b


@pytest.mark.parametrize("name", ["fp32 scales", "biases of other strides", "words of another stride"])
@pytest.mark.parametrize("side", ["keys", "values"])
def test_a_cache_given_other_buffers(monkeypatch, side, name):
    """Buffers the cache did not allocate (restored, views of one's own): what the kernel does not take is written by the
    torch ops, as it was."""
    from dspark_rocm.kv_cache import QuantizedKVCache

    monkeypatch.setattr(ops, "eager_inference", lambda *ts: True)

    def kernel(keys, values, k_rows, v_rows, *, bits, group_size):
        raise AssertionError("buffers that the kernel refuses")

    monkeypatch.setattr(ops, "quantize_kv", kernel)
    x = torch.randn(1, 2, 5, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    c, want = (QuantizedKVCache(1, 2, 128, bits=8, device="cpu") for _ in range(2))
    setattr(c, side, _other_buffers(name, getattr(c, side)))
    got = c.update_and_fetch(x, x + 1)
    monkeypatch.setattr(ops, "eager_inference", lambda *ts: False)
    for g, w in zip(got, want.update_and_fetch(x, x + 1)):
        assert all(torch.equal(a.to(b.dtype), b) for a, b in zip(g, w))


def test_a_cache_of_its_own_buffers_goes_by_the_kernel(monkeypatch):
    from dspark_rocm.kv_cache import QuantizedKVCache

    monkeypatch.setattr(ops, "eager_inference", lambda *ts: True)
    calls = []
    monkeypatch.setattr(ops, "quantize_kv", lambda *a, **k: calls.append(a))
    x = torch.zeros(1, 2, 5, 128, dtype=torch.bfloat16)
    c = QuantizedKVCache(1, 2, 128, bits=4, device="cpu")
    c.update_and_fetch(x, x)
    c.keys = _other_buffers("uint32 words", c.keys)
    c.values = _other_buffers("uint32 words", c.values)
    c.update_and_fetch(x, x)
    assert len(calls) == 2
