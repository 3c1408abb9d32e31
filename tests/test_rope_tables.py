"""CPU: the rotary tables against their formulas, the torch rotation against the closed form, refusals."""

from __future__ import annotations

import math

import pytest
import torch

from dspark_rocm import _lib, ops, rope
from dspark_rocm.model import ModelArgs, rope as model_rope


def test_default_and_linear():
    f, s = rope.frequencies(8, 1e4)
    assert s == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.equal(rope.frequencies(8, 1e4, {"type": "linear", "factor": 4.0})[0], f / 4)
    assert torch.equal(rope.frequencies(8, 1e4, {"rope_type": "default"})[0], f)


def test_llama3():
    cfg = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
    f, s = rope.frequencies(128, 5e5, cfg)
    plain = rope.frequencies(128, 5e5)[0]
    for a, b in zip(f.tolist(), plain.tolist()):
        wave = 2 * math.pi / b
        if wave < 8192 / 4:
            want = b
        elif wave > 8192:
            want = b / 8
        else:
            t = (8192 / wave - 1) / 3
            want = (1 - t) * b / 8 + t * b
        assert abs(a - want) <= 1e-14 * want
    assert s == 1.0 and f[0] == plain[0] and f[-1] == plain[-1] / 8


def test_yarn():
    cfg = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)
    f, s = rope.frequencies(128, 1e6, cfg)
    plain = rope.frequencies(128, 1e6)[0]
    assert s == 0.1 * math.log(4.0) + 1.0
    r = (f / plain).tolist()
    assert r == sorted(r, reverse=True) and r[0] == 1.0 and r[-1] == 0.25
    # the first slowed pair is the one after 32 turns over 32768 positions, the last mixed one before 1 turn
    turns = (32768 * plain / (2 * math.pi)).tolist()
    assert all(x == 1.0 for x, t in zip(r, turns) if t > 32 * 1.25) and all(x == 0.25 for x, t in zip(r, turns) if t < 0.8)
    assert rope.frequencies(128, 1e6, {**cfg, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("dims,base,scaling", [
    (7, 1e4, None), (0, 1e4, None), (8, 0.0, None), (8, 1e4, dict(type="linear")), (8, 1e4, dict(type="linear", factor=0)),
    (8, 1e4, dict(type="longrope", factor=2.0)), (8, 1e4, dict(type="llama3", factor=2.0)),
    (8, 1e4, dict(type="yarn", factor=2.0)), (8, 1.0, dict(type="yarn", factor=2.0, original_max_position_embeddings=10)),
    (8, 1e4, dict(type="llama3", factor=2.0, low_freq_factor=4.0, high_freq_factor=4.0, original_max_position_embeddings=10))])
def test_refused_tables(dims, base, scaling):
    with pytest.raises(ValueError):
        rope.frequencies(dims, base, scaling)


@pytest.mark.parametrize("inter", [False, True])
def test_rotate_unit_vectors(inter):
    f, _ = rope.frequencies(8, 1e4)
    for i in range(4):
        at, to = (2 * i, 2 * i + 1) if inter else (i, i + 4)
        x = torch.zeros(1, 1, 1, 12)
        x[..., at] = 1.0
        x[..., 8:] = 3.0
        for p in (0, 1, 17, 123456):
            y = rope.rotate(x, f, p, interleaved=inter, scale=2.0)[0, 0, 0]
            want = torch.zeros(12)
            want[8:] = 3.0
            want[at], want[to] = 2 * math.cos(p * float(f[i])), 2 * math.sin(p * float(f[i]))
            assert (y - want).abs().max() <= 4 * 2.0 ** -24
    x = torch.randn(2, 3, 5, 8, requires_grad=True)                 # autograd follows it
    rope.rotate(x, f, torch.arange(10).view(2, 5), interleaved=inter).square().sum().backward()
    assert torch.allclose(x.grad, 2 * x.detach(), atol=1e-5)        # a rotation keeps lengths


def test_rotate_is_the_model_rotation_at_near_positions():
    x = torch.randn(1, 2, 6, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    d = (rope.rotate(x, rope.frequencies(64, 1e6)[0], 5).double() - model_rope(x, 5, 1e6).double()).abs()
    assert float(d.max()) <= 2.0 ** -7 * float(x.abs().max()) * 2 ** 0.5    # one bf16 rounding apart at most


def test_which_targets_need_a_table():
    base = dict(hidden_size=64, num_hidden_layers=1, intermediate_size=64, num_attention_heads=1, num_key_value_heads=1,
                head_dim=64, vocab_size=64)
    assert ModelArgs(**base).fused_rope and ModelArgs(**base, rope_dims=64, rope_scaling={"type": "default"}).fused_rope
    for kw in (dict(rope_dims=32), dict(rope_traditional=True), dict(rope_scaling=dict(type="linear", factor=2.0))):
        a = ModelArgs(**base, **kw)
        assert not a.fused_rope and a.rope_table("cpu")[0].numel() == (kw.get("rope_dims") or 64) // 2
        hash(a)


@pytest.mark.parametrize("change,status", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(freqs=None), -1), (dict(k=None), -1), (dict(dtype=3), -6), (dict(D=1), -2),
    (dict(D=1026), -2), (dict(dims=258, D=512), -2), (dict(dims=66), -2), (dict(dims=7), -2), (dict(dims=0), -2), (dict(B=0), -2),
    (dict(L=0), -2), (dict(B=1 << 13, L=1 << 13), -2), (dict(Hq=0), -2), (dict(Hk=-1), -2), (dict(Hq=5000), -2),
    (dict(q=(1 << 20) + 1), -3)])
def test_rope_refuses(change, status):
    """Refused on the host: the pointers are never followed."""
    fake = 1 << 20
    a = dict(dtype=0, q=fake, Hq=2, k=fake, Hk=1, B=1, L=3, D=64, dims=64, freqs=fake, out=fake)
    a.update(change)
    six = (64,) * 6
    st = _lib.load().dspark_rope(ops._ROPE_ARGS.pack(a["dtype"], a["q"] or 0, a["out"] or 0, *six, a["Hq"], a["k"] or 0, fake, *six,
                                                     a["Hk"], a["B"], a["L"], a["D"], a["dims"], 0, a["freqs"] or 0, 1.0, 0, 0, 0,
                                                     0, 0), None)
    assert _lib.load().dspark_rope(None, None) == -1
    assert st == status and _lib.load().dspark_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(bits=3), -6), (dict(group=32), -6), (dict(x_dtype=5), -6), (dict(c_dtype=2), -6), (dict(D=96), -2), (dict(D=0), -2),
    (dict(D=8192), -2), (dict(B=0), -2), (dict(B=300, H=300), -2), (dict(T=0), -2), (dict(T=1 << 40), -2), (dict(x=0), -1),
    (dict(w=0), -1), (dict(x=(1 << 20) + 1), -3), (dict(w=(1 << 20) + 2), -3)])
@pytest.mark.parametrize("write", [True, False])
def test_kv_refuses(change, status, write):
    fake = 1 << 20
    a = dict(x_dtype=0, c_dtype=0, x=fake, w=fake, B=1, H=2, T=5, D=64, bits=8, group=64)
    a.update(change)
    lib = _lib.load()
    call = lib.dspark_kv_quantize if write else lib.dspark_kv_dequantize
    side = lambda x, w: (x, 64, 64, 64, w, fake, fake, 64, 64, 64, 64, 64, 64)
    st = call(ops._KV_ARGS.pack(a["x_dtype"], a["c_dtype"], a["B"], a["H"], a["T"], a["D"], a["bits"], a["group"],
                                *side(a["x"], a["w"]), *side(fake, fake)), None)
    assert call(None, None) == -1
    assert st == status and lib.dspark_last_error()


def test_host_checks():
    x = torch.zeros(1, 1, 1, 64)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.rope(x, None, rope.frequencies(64, 1e4)[0], 0)
    w, s = torch.zeros(1, 1, 1, 16, dtype=torch.int32), torch.zeros(1, 1, 1, 1, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.quantize_kv(x, x, (w, s, s), (w, s, s), bits=8)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.dequantize_kv((w, s, s), (w, s, s), bits=8)


@pytest.mark.parametrize("extra", [dict(mscale=1.0), dict(mscale_all_dim=0.7), dict(truncate=False)])
def test_yarn_settings_that_are_not_taken(extra):
    with pytest.raises(ValueError, match="not taken"):
        rope.frequencies(64, 1e4, dict(type="yarn", factor=4.0, original_max_position_embeddings=4096, **extra))


def test_rows_past_one_launch():
    """A workgroup a row: 2^24 rows are 2^32 threads."""
    fake, six = 1 << 20, (64,) * 6
    pack = lambda B, L: ops._ROPE_ARGS.pack(0, fake, fake, *six, 1, 0, 0, *six, 0, B, L, 64, 64, 0, fake, 1.0, 0, 0, 0, 0, 0)
    for B, L in ((1, 1 << 24), (1 << 24, 1), (1 << 12, 1 << 12)):
        assert _lib.load().dspark_rope(pack(B, L), None) == -2


@pytest.mark.parametrize("inter", [False, True])
def test_rotate_in_64_bits(inter):
    """fp64 tensors are rotated in fp64: within the angle's and four operations' roundings; gradients and tangents
    against differences."""
    f, _ = rope.frequencies(8, 1e4)
    x = torch.randn(2, 3, 5, 12, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    pos = torch.arange(10).view(2, 5)
    y = rope.rotate(x, f, pos, interleaved=inter, scale=1.25)
    a, b = (x[..., 0:8:2], x[..., 1:8:2]) if inter else (x[..., :4], x[..., 4:8])
    z = torch.complex(a, b) * torch.polar(torch.full((), 1.25, dtype=torch.float64), pos[:, None, :, None] * f)
    want = torch.stack([z.real, z.imag], -1).flatten(-2) if inter else torch.cat([z.real, z.imag], -1)
    assert torch.equal(y[..., 8:], x[..., 8:]) and (y[..., :8] - want).abs().max() <= 8 * 2.0 ** -52 * 1.25 * float(x.abs().max())
    assert torch.autograd.gradcheck(lambda t: rope.rotate(t, f, pos, interleaved=inter), x.requires_grad_(), check_forward_ad=True)
