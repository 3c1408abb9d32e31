"""CPU: the sampling oracle against hand-worked rows, and the refusals of the sampling entry points."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sampling_ref as ref


def test_weights_by_hand():
    x = np.log([4.0, 1.0, 2.0, 1.0])
    np.testing.assert_allclose(ref.probs(x), [0.5, 0.125, 0.25, 0.125], rtol=1e-15)
    np.testing.assert_allclose(ref.probs(x, top_k=3), [4 / 7, 1 / 7, 2 / 7, 0], rtol=1e-15)     # the tie by index
    np.testing.assert_allclose(ref.probs(x, temperature=0.5), np.array([16, 1, 4, 1]) / 22, rtol=1e-14)
    np.testing.assert_array_equal(ref.probs(np.zeros(6), top_p=0.5) > 0, [1, 1, 1, 0, 0, 0])    # 3 are half already
    np.testing.assert_array_equal(ref.probs(np.zeros(6), top_k=4, top_p=0.6) > 0, [1, 1, 1, 0, 0, 0])
    np.testing.assert_array_equal(ref.probs([-np.inf, np.nan, 3.0, np.inf]), [0, 0, 0, 1])
    np.testing.assert_array_equal(ref.probs([-np.inf, np.nan]), [0, 0])


def test_committed_token_follows_the_target():
    """Over every draft and a fine grid of both random numbers, a one-draft round commits the target's p."""
    r = np.random.default_rng(3)
    V, grid = 5, 400
    x = r.standard_normal((1, 2, V))
    q = r.dirichlet(np.ones(V))
    p = ref.probs(x[0, 0], top_p=0.9)
    got = np.zeros(V)
    us = (np.arange(grid) + 0.5) / grid
    for d in range(V):
        for u in us:
            accepted = u * q[d] < p[d]
            if accepted:
                got[d] += q[d] / grid
                continue
            for last in us[::20]:
                n, tokens, _ = ref.verify(x, np.array([[d]]), np.array([[u, last]]), q[None, None], top_p=0.9)
                assert n[0] == 0
                got[tokens[0, 0]] += q[d] / grid / len(us[::20])
    assert np.abs(got - p).max() < 0.03         # the 20 strata of the second number


def _lib():
    from dspark_rocm import _lib

    return _lib.load()


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -6), (dict(rows=0), -2), (dict(rows=65536), -2), (dict(V=0), -2), (dict(V=524281), -2), (dict(ld=99), -2),
    (dict(temperature=0.0), -1), (dict(temperature=-1.0), -1), (dict(temperature=float("nan")), -1),
    (dict(temperature=float("inf")), -1), (dict(top_k=-1), -1), (dict(top_p=0.0), -1), (dict(top_p=1.5), -1),
    (dict(top_p=float("nan")), -1), (dict(logits=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(nbytes=-1), -4),
    (dict(ws=(1 << 20) + 16), -3), (dict(logits=(1 << 20) + 1), -3), (dict(out=(1 << 20) + 2), -3)])
def test_sampling_probs_refuses(change, status):
    """Refused on the host: the pointers are never followed."""
    from dspark_rocm import ops

    lib = _lib()
    fake = 1 << 20
    a = dict(dtype=0, logits=fake, ld=100, rows=3, V=100, temperature=1.0, top_k=0, top_p=1.0, out=fake, ws=fake, nbytes=0)
    a.update(change)
    need = lib.dspark_sampling_workspace(a["rows"], a["V"], 0)
    assert (need == 0) == (status == -2 and "ld" not in change)
    st = lib.dspark_sampling_probs(ops._PROBS_ARGS.pack(a["dtype"], a["logits"] or 0, a["ld"], a["rows"], a["V"], a["temperature"],
                                                        a["top_k"], a["top_p"], a["out"] or 0, 100, a["ws"] or 0,
                                                        max(need + a["nbytes"], 0)), None)
    assert lib.dspark_sampling_probs(None, None) == -1
    assert st == status and lib.dspark_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), -6), (dict(B=0), -2), (dict(m=-1), -2), (dict(m=256), -2), (dict(V=0), -2), (dict(B=65535), -2),
    (dict(draft=None), -1), (dict(u=None), -1), (dict(n=None), -1), (dict(tokens=None), -1), (dict(px=None), -1),
    (dict(temperature=0.0), -1), (dict(top_p=-0.1), -1), (dict(ld=-5), -2), (dict(nbytes=-1), -4), (dict(u=(1 << 20) + 2), -3),
    (dict(u=(1 << 20) + 4, f64=1), -3)])
def test_speculative_verify_refuses(change, status):
    from dspark_rocm import ops

    lib = _lib()
    fake = 1 << 20
    a = dict(dtype=0, ld=100, B=2, m=3, V=100, draft=fake, u=fake, f64=0, temperature=1.0, top_p=1.0, n=fake, tokens=fake,
             px=fake, nbytes=0)
    a.update(change)
    need = lib.dspark_sampling_workspace(a["B"] * (a["m"] + 1), a["V"], max(a["B"], 0))
    st = lib.dspark_speculative_verify(ops._VERIFY_ARGS.pack(
        a["dtype"], fake, 4 * a["ld"], a["ld"], a["B"], a["m"], a["V"], a["draft"] or 0, 0, 0, 0, 0, a["u"] or 0, a["f64"],
        a["temperature"], 0, a["top_p"], a["n"] or 0, a["tokens"] or 0, a["px"] or 0, fake, max(need + a["nbytes"], 0)), None)
    assert lib.dspark_speculative_verify(None, None) == -1
    assert st == status and lib.dspark_last_error()


def test_host_checks():
    from dspark_rocm import ops

    x = torch.zeros(2, 3, 10, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.sampling_probs(x)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.speculative_verify(x, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3))
    for bad in (dict(temperature=0), dict(temperature=-1.0), dict(top_k=-3), dict(top_p=0.0), dict(top_p=1.01)):
        with pytest.raises(ValueError):
            ops.check_sampler(**{**dict(temperature=1.0, top_k=0, top_p=1.0), **bad})
    assert ops.sampling_workspace_bytes(16, 151936, 1) > 16 * 297 * 12


@pytest.mark.parametrize("at", [7, 8, 11, 17, 18, 19])
def test_speculative_verify_refuses_odd_addresses(at):
    """Each array of 4-byte elements (field ``at`` of the struct) two bytes off: refused on the host."""
    from dspark_rocm import ops

    lib = _lib()
    fake = 1 << 20
    fields = [0, fake, 400, 100, 2, 3, 100, fake, fake, 300, 100, fake, fake, 0, 1.0, 0, 1.0, fake, fake, fake, fake,
              lib.dspark_sampling_workspace(8, 100, 2)]
    fields[at] = fake + 2
    assert lib.dspark_speculative_verify(ops._VERIFY_ARGS.pack(*fields), None) == -3


@pytest.mark.parametrize("rows,V,per", [(1, 151936, 1), (16, 151936, 16), (20, 50257, 4), (256, 151936, 8), (3, 1000, 1)])
def test_workspace_of_a_sampler(rows, V, per):
    """Only what cuts by a mass, or by a top_k that is counted, needs room for counts; a call with less is refused."""
    from dspark_rocm import ops

    lib = _lib()
    fake = 1 << 20
    for seqs in (0, rows // per):
        most = lib.dspark_sampling_workspace(rows, V, seqs)
        for k, p in ((0, 1.0), (1, 1.0), (20, 0.9), (128, 0.5), (V, 1.0), (1 << 31, 1.0), (0, 0.9), (129, 1.0), (700, 0.9), (V, 0.9)):
            need = lib.dspark_sampling_workspace_for(rows, V, seqs, k, p)
            counted = (k > 128 and k < V) or (p < 1.0 and (k == 0 or k >= V))
            groups = min(256 // rows, (-(-(V + 7) // 512) + 15) // 16, 8)
            assert most - need == (0 if counted or groups < 2 else rows * groups * 61440 * 2)
            assert need == ops.sampling_workspace_bytes(rows, V, seqs, k, p)
            if seqs:
                fields = [0, fake, per * V, V, seqs, per - 1, V, fake, 0, 0, 0, 0, fake, 0, 1.0, k, p, fake, fake, fake, fake, need - 1]
                assert lib.dspark_speculative_verify(ops._VERIFY_ARGS.pack(*fields), None) == -4
            else:
                assert lib.dspark_sampling_probs(ops._PROBS_ARGS.pack(0, fake, V, rows, V, 1.0, k, p, fake, V, fake, need - 1), None) == -4
    assert ops.sampling_workspace_bytes(rows, V) == lib.dspark_sampling_workspace(rows, V, 0)
    assert lib.dspark_sampling_workspace_for(0, V, 0, 0, 1.0) == 0 and lib.dspark_sampling_workspace_for(rows, 524281, 0, 0, 1.0) == 0
