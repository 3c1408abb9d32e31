"""CPU: the oracle of paged caches and token scores against closed forms."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import paged_ref


def test_e4m3_is_torchs():
    x = torch.cat([torch.linspace(-470, 470, 40001), torch.linspace(-0.04, 0.04, 4001), torch.tensor([464.0, 464.01, float("nan"), 2.0 ** -10, 2.0 ** -10 * 1.01])])
    want = x.to(torch.float8_e4m3fn).double().numpy()
    got = paged_ref.e4m3(x.double().numpy())
    np.testing.assert_array_equal(got, want)


def test_rotation_keeps_lengths_and_turns_by_the_angle():
    x = np.zeros((2, 1, 8))
    x[:, 0, 1] = 3.0
    f = np.array([1.0, 0.25, 0.1])
    y = paged_ref.rotate(x, [0, 5], f)
    np.testing.assert_array_equal(y[0], x[0])
    assert abs(y[1, 0, 1] - 3 * math.cos(1.25)) < 1e-6 and abs(y[1, 0, 4] - 3 * math.sin(1.25)) < 1e-6
    z = paged_ref.rotate(x, [0, 5], f, interleaved=True)
    assert abs(z[1, 0, 0] + 3 * math.sin(5)) < 1e-6 and abs(z[1, 0, 1] - 3 * math.cos(5)) < 1e-6


def test_exponents():
    e = paged_ref.exponent
    assert e(np.array([448.0, -1]), None) == 0 and e(np.array([449.0]), None) == 1 and e(np.array([-224.0]), None) == -1
    assert e(np.array([0.0]), None) == -110 and e(np.array([1.0, np.inf, np.nan]), -20) == -8 and e(np.array([1.0]), 3) == 3


def test_pages_grow_and_start_again():
    p = paged_ref.Pages(np.zeros((2, 1, 4, 2)), np.zeros((2, 1)))
    table = np.array([[1]])
    paged_ref.append(p, np.full((1, 1, 2), 0.3), table, [0, 1], [1])
    assert p.exps[1, 0] == -10 and abs(p.values[1, 0, 0, 0] - 0.3) <= 0.3 / 16
    paged_ref.append(p, np.full((1, 1, 2), 448.0), table, [0, 1], [2])
    assert p.exps[1, 0] == 0 and p.values[1, 0, 1, 0] == 448.0 and abs(p.values[1, 0, 0, 0] - 0.3) <= 0.3 / 16 * 2
    paged_ref.append(p, np.full((1, 1, 2), 0.3), table, [0, 1], [1])
    assert p.exps[1, 0] == -10
    paged_ref.append(p, np.full((6, 1, 2), 1.0), table, [0, 6], [3])        # three rows before the first position
    assert (p.values[1, 0, :3] == 1.0).all()
    before = p.values.copy()
    paged_ref.append(p, np.full((1, 1, 2), 1.0), np.array([[2]]), [0, 1], [1])
    paged_ref.append(p, np.full((1, 1, 2), 1.0), table, [0, 1], [5])
    np.testing.assert_array_equal(p.values, before)


def test_attention_closed_forms():
    g = np.random.default_rng(0)
    k, v = paged_ref.Pages(np.zeros((3, 2, 4, 8))), paged_ref.Pages(g.standard_normal((3, 2, 4, 8)))
    q = g.standard_normal((4, 4, 8))
    table = np.array([[2, 0], [1, -1]])
    o = paged_ref.attention(q, k, v, table, [0, 2, 3], [6, 3], 1.0)
    flat = np.concatenate([v.values[2], v.values[0]], 1)
    for h in range(4):
        np.testing.assert_allclose(o[0, h], flat[h // 2, :5].mean(0), rtol=1e-12)      # equal scores: the mean of what a row sees
        np.testing.assert_allclose(o[1, h], flat[h // 2, :6].mean(0), rtol=1e-12)
        np.testing.assert_allclose(o[2, h], v.values[1, h // 2, :3].mean(0), rtol=1e-12)
    assert np.isnan(o[3]).all()
    o = paged_ref.attention(q, k, v, table, [0, 2, 3], [1, 5], 1.0, causal=False)
    np.testing.assert_allclose(o[0, 0], v.values[2, 0, 0], rtol=1e-12)
    np.testing.assert_allclose(o[2, 0], v.values[1, 0].mean(0), rtol=1e-12)            # the page that is not there is not seen
    assert not paged_ref.attention(q, k, v, table, [0, 2, 3], [1, 5], 1.0)[0].any()    # before the first position


def test_logprobs_closed_forms():
    x = np.log(np.array([0.5, 0.25, 0.125, 0.125]))
    lp, h, ids, best = paged_ref.logprobs(x, 2, 3)
    assert abs(lp - math.log(0.125)) < 1e-12 and abs(h - 1.75 * math.log(2)) < 1e-12
    assert ids.tolist() == [0, 1, 2] and abs(best[1] - math.log(0.25)) < 1e-12
    assert abs(paged_ref.logprobs(x, 0, temperature=0.5)[0] - math.log(0.25 / (0.25 + 0.0625 + 2 / 64))) < 1e-12
    lp, h, ids, best = paged_ref.logprobs([np.nan, np.inf, 1.0, np.inf], 3, 4)
    assert abs(lp + math.log(2)) < 1e-12 and abs(h - math.log(2)) < 1e-12 and ids.tolist() == [1, 3, 2, 0] and best[2] == -np.inf
    lp, h, ids, best = paged_ref.logprobs([-np.inf, np.nan], 0, 2)
    assert lp == -np.inf and h == 0 and ids.tolist() == [0, 1] and (best == -np.inf).all()
    assert paged_ref.logprobs([1.0, 2.0], 7)[0] == -np.inf


def test_attention_of_many_keys_is_the_loops():
    from tests._paged import attention

    g = np.random.default_rng(1)
    k, v = (paged_ref.Pages(g.standard_normal((6, 2, 4, 8))) for _ in range(2))
    q = g.standard_normal((9, 4, 8))
    table = np.array([[2, 0, 5], [1, -1, 7], [3, 4, 0]])
    for starts, lens in (([0, 2, 5, 8], [6, 12, 5]), ([0, 5, 5, 6], [3, 12, 99]), ([0, 1, 99, 6], [1, 1, 1])):
        for causal in (True, False):
            np.testing.assert_allclose(attention(q, k, v, table, starts, lens, 0.3, causal)[0],
                                       paged_ref.attention(q, k, v, table, starts, lens, 0.3, causal), rtol=1e-12, atol=1e-14)
