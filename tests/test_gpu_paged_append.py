"""GPU: ops.paged_append and ops.paged_read against the oracle's rules.

The rule names every rounding but that of the angle's cosine and sine to fp32: values are the same bits, but where the
64-bit functions of the two sides, each within 2^-50 of the true one, round to different fp32 neighbours (one in 2^25)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref
from tests._paged import DT, exps, host, ints, make_pages, make_table, oracle_pages, starts_of, typed

pytestmark = pytest.mark.gpu


def run(dev, dtype, bits, Hq, Hk, D, P, lens, rows, dims, inter, seed=0, positions=None, scale=1.0, behind=0, views=False):
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(seed)
    T = sum(rows) + behind
    dt = DT[dtype]
    pool = sum(-(-max(n, 0) // P) for n in lens) + 3
    kp, vp = (make_pages(g, pool, Hk, P, D, dt, bits, dev) for _ in range(2))
    table = make_table(g, lens, P, pool, dev)
    starts, lens_t = starts_of(rows, dev), ints(lens, dev)
    x = torch.randn(T, (Hq + 2 * Hk) * D, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    q, k, v = (t.unflatten(1, (-1, D)) for t in x.to(dt).to(dev).split([Hq * D, Hk * D, Hk * D], 1))
    if not views:
        q, k, v = (t.clone() for t in (q, k, v))
    freqs = rope.frequencies(dims, 1e4, device=dev)[0] if dims else None
    want_k, want_v = oracle_pages(kp), oracle_pages(vp)
    pos = np.zeros(T)
    for b, s0, n, p0 in paged_ref.sequences(table.cpu().numpy(), starts.cpu().numpy(), lens, T):
        pos[s0:s0 + n] = np.arange(p0, p0 + n)
    at = pos if positions is None else positions.cpu().numpy()
    turn = lambda t: paged_ref.rotate(host(t), at, host(freqs), inter, scale, typed(dt)) if dims else host(t)
    for pages, rows_ in ((want_k, turn(k)), (want_v, host(v))):
        paged_ref.append(pages, rows_, table.cpu().numpy(), starts.cpu().numpy(), lens)
    yq = ops.paged_append(k, v, kp, vp, table, starts, lens_t, q=q, freqs=freqs, positions=positions, interleaved=inter, scale=scale)
    got_k, got_v = oracle_pages(kp), oracle_pages(vp)
    for got, want in ((got_k, want_k), (got_v, want_v)):
        np.testing.assert_array_equal(got.values, want.values)
        if bits == 8:
            np.testing.assert_array_equal(got.exps, want.exps)
    n = sum(rows)
    np.testing.assert_array_equal(host(yq)[:n], turn(q)[:n])
    assert not yq[n:].any()
    return kp, vp, table, starts, lens_t


SHAPES = [  # Hq, Hk, D, P, lens, rows
    (1, 1, 64, 16, [1], [1]),
    (32, 8, 128, 64, [1000], [1]),
    (4, 2, 128, 16, [16, 17, 33, 1, 15, 0, 40], [1, 1, 1, 1, 3, 0, 40]),
    (9, 3, 64, 32, [70, 33, 64], [70, 2, 33]),
    (6, 1, 256, 128, [300, 129], [290, 1]),
    (2, 2, 256, 64, [65, 64, 128], [2, 64, 65]),
]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_append(dev, shape, dtype, bits, inter):
    Hq, Hk, D, P, lens, rows = shape
    run(dev, dtype, bits, Hq, Hk, D, P, lens, rows, D if not inter else D // 2, inter, views=True)


@pytest.mark.parametrize("bits", [16, 8])
def test_long_and_many(dev, bits):
    run(dev, "bf16", bits, 8, 2, 128, 64, [700, 1300], [600, 555], 128, False)
    run(dev, "bf16", bits, 4, 2, 64, 16, [1 + i % 37 for i in range(150)], [1 + (i % 5 if i % 37 > 6 else 0) for i in range(150)], 64, False)


@pytest.mark.parametrize("bits", [16, 8])
def test_positions_scale_and_no_rotation(dev, bits):
    g = torch.Generator().manual_seed(5)
    for p in (torch.randint(0, 1 << 30, (9,), generator=g), torch.randint(-99, 1 << 20, (9,), generator=g).to(torch.int32),
              torch.randint(0, 1 << 20, (18,), generator=g)[::2]):
        run(dev, "bf16", bits, 4, 2, 128, 16, [20, 7], [5, 4], 96, False, positions=p.to(dev), scale=1.25)
    run(dev, "f16", bits, 4, 2, 128, 16, [20, 7], [5, 4], 0, False, behind=3)


@pytest.mark.parametrize("bits", [16, 8])
def test_rows_that_have_no_place(dev, bits):
    """Rows before the first position, past the table, in pages that are not the pool's, of sequences whose rows are not the
    call's: nothing is written for them."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(1)
    Hk, D, P, pool, T = 2, 64, 16, 6, 40
    for table, starts, lens in (([[0, 1]], [0, 40], [40]), ([[0, 1, 2]], [0, 20], [7]), ([[3, 9, 2]], [0, 40], [40]),
                                ([[3, -1, 2]], [0, 40], [44]), ([[1, 2, 3]], [5, 99], [48]), ([[1, 2, 3]], [9, 3], [48]),
                                ([[1, 2, 3]], [-4, 3], [48]), ([[1, 2, 3], [4, 5, 0]], [0, 7, 7], [48, 20]),
                                ([[1, 2, 3]], [0, 4], [-5]), ([[1, 2, 3]], [0, 4], [2 ** 31 - 1]),
                                ([[2 ** 31 - 1, -2 ** 31, 3]], [0, 40], [48])):
        kp, vp = (make_pages(g, pool, Hk, P, D, torch.bfloat16, bits, dev) for _ in range(2))
        k, v = (torch.randn(T, Hk, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
        want_k, want_v = oracle_pages(kp), oracle_pages(vp)
        for pages, x in ((want_k, k), (want_v, v)):
            paged_ref.append(pages, host(x), np.array(table), starts, lens)
        assert ops.paged_append(k, v, kp, vp, ints(table, dev), ints(starts, dev), ints(lens, dev)) is None
        np.testing.assert_array_equal(oracle_pages(kp).values, want_k.values)
        np.testing.assert_array_equal(oracle_pages(vp).values, want_v.values)


def test_scales_grow_and_start_again(dev):
    """Token after token into one page: the scale only grows, earlier codes follow it; the next page, and a page that is used
    again from its first row, start anew. All zeros; values that are not finite; the largest and smallest."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(2)
    Hk, D, P = 2, 64, 16
    for dtype in (torch.bfloat16, torch.float16):
        kp, vp = (make_pages(g, 2, Hk, P, D, dtype, 8, dev) for _ in range(2))
        want_k, want_v = oracle_pages(kp), oracle_pages(vp)
        table, starts = ints([[1, 0]], dev), ints([0, 1], dev)
        size = [0.0, 1e-3, 1.0, 0.1, 60.0, 7.0, 1e4, 3.0, 1e-7, 448.0, 449.0, 6e4, 1.0, 2.0, 3.0, 4.0, 0.5, 1e-6, 2.0] + [1.0] * 5
        for i, s in enumerate(size):
            n = i + 1 if i < 19 else i - 18         # the last ones: the sequence starts again
            k, v = ((torch.randn(1, Hk, D, generator=g) * s).to(dtype) for _ in range(2))
            if i == 5:
                k[0, 0, 3], k[0, 1, 7], v[0, 0, 0] = float("inf"), float("nan"), -float("inf")
            if i == 7 and dtype is torch.bfloat16:
                k[0, 0, 0], v[0, 1, 1] = 3.3e38, -1e-38
            for pages, x in ((want_k, k), (want_v, v)):
                paged_ref.append(pages, host(x), table.cpu().numpy(), [0, 1], [n])
            ops.paged_append(k.to(dev), v.to(dev), kp, vp, table, starts, ints([n], dev))
            for got, want in ((kp, want_k), (vp, want_v)):
                np.testing.assert_array_equal(exps(got[1]), want.exps, err_msg=f"{i}")
                np.testing.assert_array_equal(oracle_pages(got).values, want.values, err_msg=f"{i}")


def test_codes_round_to_nearest_even(dev):
    """Every bf16 value up to 448: the codes of torch's conversion."""
    from dspark_rocm import ops

    x = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[x <= 448]
    x = torch.cat([x, -x])
    D, P = 64, 128
    rows = (x.numel() + D - 2) // (D - 1)
    k = torch.full((rows * (D - 1),), 0.0)
    k[:x.numel()] = x
    k = torch.cat([k.view(rows, D - 1), torch.full((rows, 1), 448.0)], 1).to(torch.bfloat16).view(rows, 1, D).to(dev)
    n = -(-rows // P)
    kp, vp = ((torch.zeros(n, 1, P, D, device=dev).to(torch.float8_e4m3fn), torch.full((n, 1), 127, dtype=torch.uint8, device=dev)
               .view(torch.float8_e8m0fnu)) for _ in range(2))
    ops.paged_append(k, k, kp, vp, torch.arange(n, dtype=torch.int32, device=dev)[None], ints([0, rows], dev), ints([rows], dev))
    assert (exps(kp[1]) == 0).all()
    want = k.float().to(torch.float8_e4m3fn).view(torch.uint8).view(rows, D)
    for p in (kp, vp):
        assert torch.equal(p[0].view(torch.uint8).view(n * P, D)[:rows], want)


@pytest.mark.parametrize("bits", [16, 8])
def test_views_and_neighbours(dev, bits):
    """Pages [pages, positions, heads, D] seen as [pages, heads, positions, D], queries rotated in place; what lies
    between, before and behind keeps its bytes."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(3)
    Hq, Hk, D, P, pool = 4, 2, 128, 16, 5
    dt = torch.bfloat16
    base = torch.randn(2, pool, P, Hk + 1, D + 16, generator=g)
    base = base.to(dt).to(dev) if bits == 16 else base.to(torch.float8_e4m3fn).to(dev)
    sc = torch.randint(110, 120, (2, pool, Hk + 2), generator=g).to(torch.uint8).to(dev)
    view = lambda i: base[i, :, :, :Hk, :D].transpose(1, 2) if bits == 16 else (base[i, :, :, :Hk, :D].transpose(1, 2),
                                                                                 sc[i, :, :Hk].view(torch.float8_e8m0fnu))
    raw = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16)
    before, sc_before = raw(base).clone(), sc.clone()
    kp, vp = view(0), view(1)
    want = [oracle_pages(kp), oracle_pages(vp)]
    x = torch.randn(7, (Hq + 2 * Hk) * D + 8, generator=g).to(dt).to(dev)
    q, k, v = (x[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, Hq), (Hq, Hq + Hk), (Hq + Hk, Hq + 2 * Hk)))
    x0, q0 = x.clone(), host(q)
    freqs = rope.frequencies(64, 1e4, device=dev)[0]
    table, lens, starts = ints([[2, 4], [0, -1]], dev), ints([19, 3], dev), ints([0, 4, 7], dev)
    pos = np.array([15, 16, 17, 18, 0, 1, 2])
    turn = lambda t: paged_ref.rotate(t, pos, host(freqs), False, 1.0, typed(dt))
    for pages, rows in zip(want, (turn(host(k)), host(v))):
        paged_ref.append(pages, rows, table.cpu().numpy(), starts.cpu().numpy(), [19, 3])
    assert ops.paged_append(k, v, kp, vp, table, starts, lens, q=q, freqs=freqs, q_out=q) is q
    np.testing.assert_array_equal(host(q), turn(q0))
    x[:, :Hq * D] = x0[:, :Hq * D]
    assert torch.equal(x, x0)
    for p, w in zip((kp, vp), want):
        np.testing.assert_array_equal(oracle_pages(p).values, w.values)
    after = raw(base).clone()
    mask = torch.zeros_like(base, dtype=torch.bool)
    for page, lo, hi in ((2, 0, 16), (4, 0, 3), (0, 0, 3)):
        mask[:, page, lo:hi, :Hk, :D] = True
    assert torch.equal(after[~mask], before[~mask])
    assert torch.equal(sc[:, :, Hk:], sc_before[:, :, Hk:]) and torch.equal(sc[:, [1, 3]], sc_before[:, [1, 3]])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [16, 8])
def test_read(dev, dtype, bits):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(4)
    for Hk, P, D, pool, ids in ((1, 16, 64, 1, [0]), (3, 32, 128, 9, [8, 0, 0, 3]), (2, 128, 256, 4, [1, -1, 4, 3])):
        kp, vp = (make_pages(g, pool, Hk, P, D, DT[dtype], bits, dev) for _ in range(2))
        k, v = ops.paged_read(kp, vp, ints(ids, dev), dtype=DT[dtype])
        for got, pages in ((k, kp), (v, vp)):
            want = typed(DT[dtype])(oracle_pages(pages).values)
            for i, p in enumerate(ids):
                np.testing.assert_array_equal(host(got[i]), want[p] if 0 <= p < pool else 0 * want[0])
    assert ops.paged_read(kp, vp, ints([], dev), dtype=DT[dtype])[0].shape == (0, 2, 128, 256)


def test_past_32_bits(dev):
    """Pages and rows that lie more than 2^32 elements into their tensors."""
    from dspark_rocm import ops

    P, D, step = 16, 64, 1 << 31
    k_buf, v_buf = (torch.zeros((2 * step + P * D,), dtype=torch.bfloat16, device=dev) for _ in range(2))
    kp, vp = (b.as_strided((3, 1, P, D), (step, P * D, D, 1)) for b in (k_buf, v_buf))
    k = torch.randn(3, 1, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(dev)
    ops.paged_append(k, -k, kp, vp, ints([[2]], dev), ints([0, 3], dev), ints([5], dev))
    assert torch.equal(kp[2, 0, 2:5], k[:, 0]) and torch.equal(vp[2, 0, 2:5], -k[:, 0]) and not kp[:2].any()
    rk, rv = ops.paged_read(kp, vp, ints([2], dev))
    assert torch.equal(rk, kp[2:]) and torch.equal(rv, vp[2:])


def test_captured_and_other_streams(dev):
    """Captured once, replayed as the lengths grow on the device; on another stream than the current one's."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(6)
    Hq, Hk, D, P = 4, 2, 64, 16
    freqs = rope.frequencies(D, 1e4, device=dev)[0]
    state = lambda: [make_pages(torch.Generator().manual_seed(9), 8, Hk, P, D, torch.bfloat16, 8, dev) for _ in range(2)]
    table, starts, lens = ints([[1, 2, 3], [7, 0, 5]], dev), ints([0, 1, 3], dev), ints([14, 30], dev)
    rows = [[torch.randn(3, h, D, generator=g).to(torch.bfloat16).to(dev) for h in (Hq, Hk, Hk)] for _ in range(5)]
    q, k, v = (t.clone() for t in rows[0])
    kp, vp = state()
    call = lambda: ops.paged_append(k, v, kp, vp, table, starts, lens, q=q, freqs=freqs)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    (kp2, vp2), lens2 = state(), lens.clone()
    for dst, src in zip((*kp, *vp), (*kp2, *vp2)):
        dst.view(torch.uint8).copy_(src.view(torch.uint8))
    for r in rows:
        for dst, src in zip((q, k, v), r):
            dst.copy_(src)
        graph.replay()
        want = ops.paged_append(r[1], r[2], kp2, vp2, table, starts, lens2, q=r[0], freqs=freqs)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for x, y in zip((*kp, *vp), (*kp2, *vp2)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        lens += 1
        lens2 += 1
