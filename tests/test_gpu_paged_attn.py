"""GPU: ops.paged_attention against attention in 64 bits (the bounds: tests/_paged.py), over masks, lengths, pages and row
counts where it can go wrong."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged_ref
from tests._paged import DT, attention, check_rows, host, ints, make_pages, make_table, oracle_pages, starts_of

pytestmark = pytest.mark.gpu


def make(g, dev, dtype, bits, Hq, Hk, D, P, lens, rows, behind=0):
    dt = DT[dtype]
    pool = sum(-(-max(n, 0) // P) for n in lens) + 2
    kp, vp = (make_pages(g, pool, Hk, P, D, dt, bits, dev) for _ in range(2))
    table = make_table(g, [max(n, 0) for n in lens], P, pool, dev)
    q = torch.randn(sum(rows) + behind, Hq, D, generator=g).to(dt).to(dev)
    return q, kp, vp, table, starts_of(rows, dev), ints(lens, dev)


def check(args, got, scale, causal=True):
    """Probabilities are two pieces of the type, 2^-16 off together; over 8-bit pages of a bf16 model prompt chunks take one fp16
    piece: half a step, 2^-11 of the probability at most."""
    q, kp, vp, table, starts, lens = args
    pieces = 2.0 ** -11 if isinstance(kp, tuple) and q.dtype is torch.bfloat16 else 2.0 ** -16
    want, tol = attention(host(q), oracle_pages(kp), oracle_pages(vp), table.cpu().numpy(), starts.tolist(), lens.tolist(), scale, causal,
                          pieces)
    check_rows(got, want, tol)


def run(dev, dtype, bits, Hq, Hk, D, P, lens, rows, seed=0, causal=True, scale=None, behind=0, **kw):
    from dspark_rocm import ops

    args = make(torch.Generator().manual_seed(seed), dev, dtype, bits, Hq, Hk, D, P, lens, rows, behind)
    scale = scale or D ** -0.5
    got = ops.paged_attention(*args, scale=scale, causal=causal, **kw)
    check(args, got, scale, causal)
    return args, got


SHAPES = [  # Hq, Hk, D, P, lens, rows
    (1, 1, 64, 16, [1], [1]),
    (32, 8, 128, 16, [129], [1]),
    (4, 2, 128, 64, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 0, 511, 512], [1, 1, 3, 16, 1, 1, 2, 1, 5, 1, 1, 0, 1, 2]),
    (8, 1, 64, 32, [700, 64, 2050], [1, 2, 1]),
    (6, 1, 256, 32, [1300, 90, 515], [5, 1, 2]),
    (24, 4, 256, 128, [1025, 16], [16, 16]),
    (9, 3, 64, 64, [1111, 3, 40], [16, 3, 7]),
    (64, 8, 128, 128, [2500], [8]),
    (2, 2, 128, 16, [640, 1000, 77], [1, 40, 77]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(dev, shape, dtype, bits, causal):
    Hq, Hk, D, P, lens, rows = shape
    run(dev, dtype, bits, Hq, Hk, D, P, lens, rows, causal=causal, max_rows=max(rows), max_len=max(lens))


@pytest.mark.parametrize("bits", [16, 8])
def test_bounds_of_the_host(dev, bits):
    """Without the host's bounds, with loose ones, with fewer rows than a sequence has; max_len cuts what lies behind it."""
    from dspark_rocm import ops

    for kw in ({}, dict(max_rows=1), dict(max_rows=999, max_len=10 ** 9), dict(max_rows=3)):
        run(dev, "bf16", bits, 4, 2, 64, 16, [900, 33, 5], [20, 1, 5], behind=2, **kw)
    args = make(torch.Generator().manual_seed(1), dev, "bf16", bits, 4, 2, 64, 32, [900, 33], [3, 1])
    got = ops.paged_attention(*args, scale=0.125, max_len=600)
    cut = (args[0], args[1], args[2], args[3][:, :19], args[4], args[5])
    check(cut, got, 0.125)


@pytest.mark.parametrize("bits", [16, 8])
def test_many_sequences(dev, bits):
    lens = [(37 * i) % 700 + 1 for i in range(150)]
    rows = [0 if i % 7 == 3 else 1 + (i % 5 == 0) for i in range(150)]
    run(dev, "bf16", bits, 4, 2, 64, 16, [max(a, b) for a, b in zip(lens, rows)], rows, max_rows=2, max_len=700)
    run(dev, "f16", bits, 2, 1, 64, 16, [1 + i % 3 for i in range(300)], [1] * 300, max_rows=1, max_len=3)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,n", [(128, 1), (128, 6), (128, 16), (256, 2), (64, 16)])
def test_long(dev, D, n, bits):
    run(dev, "bf16", bits, 4, 1, D, 128, [20011, 4500, 64], [n, 1, n], max_rows=n, max_len=20011)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
def test_rows_that_see_nothing(dev, bits, causal):
    """More rows than positions, pages that are not the pool's, sequences that do not fit the call, lengths of zero and less,
    rows of no sequence."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(2)
    D, P, pool, T = 64, 16, 6, 24
    for table, starts, lens in (([[0, 1]], [0, 24], [20]), ([[0, 1, 2]], [0, 20], [7]), ([[3, 9, 2]], [0, 24], [40]),
                                ([[-1, -1, -1]], [0, 3], [44]), ([[1, -7, 3]], [2, 5], [48]), ([[1, 2, 3]], [5, 99], [48]),
                                ([[1, 2, 3]], [9, 3], [48]), ([[1, 2, 3]], [-4, 3], [48]), ([[1, 2, 3], [4, 5, 0]], [0, 7, 7], [48, 20]),
                                ([[1, 2, 3]], [0, 4], [-5]), ([[1, 2, 3]], [0, 4], [0]), ([[1, 2, 3]], [0, 4], [2 ** 31 - 1]),
                                ([[2 ** 31 - 1, -2 ** 31, 3]], [0, 4], [48]), ([[1] * 50], [0, 2], [800])):
        kp, vp = (make_pages(g, pool, 2, P, D, torch.bfloat16, bits, dev) for _ in range(2))
        q = torch.randn(T, 4, D, generator=g).to(torch.bfloat16).to(dev)
        args = (q, kp, vp, ints(table, dev), ints(starts, dev), ints(lens, dev))
        got = ops.paged_attention(*args, scale=0.2, causal=causal)
        check(args, got, 0.2, causal)
        out = torch.full_like(q, 7.0)
        assert ops.paged_attention(*args, scale=0.2, causal=causal, out=out) is out
        none = np.isnan(paged_ref.attention(host(q), oracle_pages(kp), oracle_pages(vp), np.array(table), starts, lens, 0.2, causal))
        none = torch.from_numpy(none).to(dev)
        assert (out[none] == 7).all() and torch.equal(out[~none], got[~none])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,L", [(1, 40), (5, 300), (4, 3000)])
def test_not_finite_where_nobody_looks(dev, dtype, bits, n, L):
    """NaN and infinities behind a sequence's end, in other pages and in keys that a row does not see leave it alone; where a
    row sees them they are what plain arithmetic gives."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(3)
    Hq, Hk, D, P = 4, 2, 64, 16
    q, kp, vp, table, starts, lens = make(g, dev, dtype, bits, Hq, Hk, D, P, [L, 17], [n, 1])
    clean = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
    data = lambda p: p[0] if bits == 8 else p
    nan, inf = float("nan"), float("inf")
    pool = data(kp).shape[0]
    used = torch.zeros(pool, P, dtype=torch.bool)
    for b, m in enumerate((L, 17)):
        for i in range(m):
            used[table[b, i // P].item(), i % P] = True
    hidden = (~used).to(dev)[:, None, :, None]
    bad = torch.full(data(kp).shape, nan, device=dev)
    if bits == 16:
        bad[..., ::3] = inf
        bad[..., 1::3] = -inf
    as_bits = lambda t: t.view(torch.uint8) if bits == 8 else t.view(torch.int16)
    spoil = lambda t, where: as_bits(t).copy_(torch.where(where, as_bits(bad.to(t.dtype)), as_bits(t)))
    for p in (kp, vp):
        spoil(data(p), hidden)
    got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
    assert torch.equal(got, clean)
    # the last position: its row alone sees it
    at = torch.zeros_like(hidden)
    at[table[0, (L - 1) // P].item(), :, (L - 1) % P] = True
    for p in (kp, vp):
        keep = data(p).clone()
        spoil(data(p), at)
        got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
        # (rows that were computed again in plain fp32 may round to the other side)
        assert torch.equal(got[n:], clean[n:])
        assert got[:n - 1].isfinite().all() and (got[:n - 1].double() - clean[:n - 1].double()).abs().max() <= 2 ** -7 * clean.double().abs().max() if n > 1 else True
        assert not got[n - 1].isfinite().any()
        data(p).copy_(keep)
    if bits == 16:
        vp[table[0, 0].item(), :, 0, 5] = inf
        vp[table[0, 0].item(), :, 0, 6] = -inf
        got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
        assert (got[:n, :, 5] == inf).all() and (got[:n, :, 6] == -inf).all()
        assert got[:n, :, :5].isfinite().all() and got[:n, :, 7:].isfinite().all() and torch.equal(got[n:], clean[n:])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_scores_and_sums(dev, dtype):
    """One key far above the rest, rising and falling scores, values near the end of the type's range."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(4)
    q, kp, vp, table, starts, lens = make(g, dev, dtype, 16, 4, 2, 64, 16, [900, 333], [2, 1])
    for order in (1, -1):
        for b, n in enumerate((900, 333)):
            for i in range(n):
                kp[table[b, i // 16].item(), :, i % 16] = q[b, 0] * (order * (i - n / 2) * 0.1)
        args = (q, kp, vp, table, starts, lens)
        check(args, ops.paged_attention(*args, scale=0.125), 0.125)
    kp.zero_()
    big = torch.finfo(DT[dtype]).max * 0.9
    vp.fill_(big)
    got = ops.paged_attention(*args, scale=0.125)
    assert torch.allclose(got.double(), vp[0, 0, 0, 0].double().expand(got.shape), rtol=2 ** -7, atol=0)


def test_views_and_streams(dev):
    """Queries and outputs as views of wider rows, pages [pages, positions, heads, D], int64 tables; another stream; the
    same bits again, with a workspace of the caller's."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(5)
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 16, 4, 2, 128, 16, [1400, 33, 700], [2, 1, 4])
    want = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    wide = torch.full((7, 6, 192), 3.0, dtype=torch.bfloat16, device=dev)
    wide[:, :4, 64:] = q
    swapped = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in (kp, vp)]
    out = torch.full((7, 9, 128), 5.0, dtype=torch.bfloat16, device=dev)
    ws = torch.full((ops.paged_attention_workspace_bytes(3, 4, 2, 128, 7, 7, table.shape[1] * 16),), 255, dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.paged_attention(wide[:, :4, 64:], *swapped, table.long(), starts.long(), lens.long(), scale=0.1, out=out[:, 2:6], workspace=ws)
    side.synchronize()
    assert torch.equal(got, want) and (out[:, :2] == 5).all() and (out[:, 6:] == 5).all()
    odd = torch.zeros(7, 4, 129, dtype=torch.bfloat16, device=dev)
    odd[..., 1:] = q
    assert torch.equal(ops.paged_attention(odd[..., 1:], kp, vp, table, starts, lens, scale=0.1), want)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured(dev, bits):
    """A captured step over device lengths: replayed as they grow, against the eager call; two graphs with a workspace each."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(6)
    q, kp, vp, table, starts, _ = make(g, dev, "bf16", bits, 8, 2, 128, 16, [2000, 800, 40], [1, 3, 2])
    lens = ints([1500, 700, 3], dev)
    call = lambda: ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1, max_rows=3)
    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for i in range(4):
        for graph, out in graphs:
            out.fill_(9.0)
        lens += 7
        q.copy_(torch.randn(q.shape, generator=g))
        for graph, _ in graphs:
            graph.replay()
        want = call()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


def test_past_32_bits(dev):
    """Pages more than 2^32 elements into their tensors."""
    from dspark_rocm import ops

    P, D, step = 16, 64, 1 << 31
    k_buf, v_buf = (torch.zeros((2 * step + P * D,), dtype=torch.bfloat16, device=dev) for _ in range(2))
    kp, vp = (b.as_strided((3, 1, P, D), (step, P * D, D, 1)) for b in (k_buf, v_buf))
    g = torch.Generator().manual_seed(0)
    kp[2], vp[2], vp[1] = (torch.randn(1, P, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(3))
    q = torch.randn(2, 1, D, generator=g).to(torch.bfloat16).to(dev)
    args = (q, kp, vp, ints([[2, 1]], dev), ints([0, 2], dev), ints([30], dev))
    got = ops.paged_attention(*args, scale=0.125)
    small = [torch.stack([p[0], p[1], p[2]]) for p in (kp, vp)]
    assert torch.equal(got, ops.paged_attention(q, *small, *args[3:], scale=0.125))
    check((q, *small, *args[3:]), got, 0.125)


@pytest.mark.parametrize("bits", [16, 8])
def test_append_then_attend(dev, bits):
    """A prompt in two chunks, then tokens one by one, for three sequences beside each other, as a server runs them: the
    same as attention over what the pages hold."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(7)
    Hq, Hk, D, P = 8, 2, 64, 16
    freqs = rope.frequencies(D, 1e4, device=dev)[0]
    kp, vp = (make_pages(g, 24, Hk, P, D, torch.bfloat16, bits, dev) for _ in range(2))
    table = torch.randperm(24, generator=g).to(torch.int32).view(3, 8).to(dev)
    lens = [0, 0, 0]
    for rows in ([33, 20, 0], [7, 0, 48], [1, 1, 1], [1, 1, 1], [4, 0, 2], [1, 1, 1]):
        lens = [a + b for a, b in zip(lens, rows)]
        T = sum(rows)
        q, k, v = (torch.randn(T, h, D, generator=g).to(torch.bfloat16).to(dev) for h in (Hq, Hk, Hk))
        starts, n = starts_of(rows, dev), ints(lens, dev)
        y = ops.paged_append(k, v, kp, vp, table, starts, n, q=q, freqs=freqs)
        args = (y, kp, vp, table, starts, n)
        check(args, ops.paged_attention(*args, scale=D ** -0.5, max_rows=max(rows)), D ** -0.5)


def test_encoder_states(dev):
    """Attention to an encoder's states of another length: appended without rotation, all of them seen."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(8)
    Hk, D, P, lens = 2, 64, 32, [150, 31]
    kp, vp = (make_pages(g, 7, Hk, P, D, torch.float16, 16, dev) for _ in range(2))
    table = make_table(g, lens, P, 7, dev)
    k, v = (torch.randn(sum(lens), Hk, D, generator=g).to(torch.float16).to(dev) for _ in range(2))
    ops.paged_append(k, v, kp, vp, table, starts_of(lens, dev), ints(lens, dev))
    q = torch.randn(9, 4, D, generator=g).to(torch.float16).to(dev)
    got = ops.paged_attention(q, kp, vp, table, ints([0, 4, 9], dev), ints(lens, dev), scale=0.2, causal=False)
    for s, e, lo in ((0, 4, 0), (4, 9, 150)):
        n = 150 if lo == 0 else 31
        kk, vv = (t[lo:lo + n].double().repeat_interleave(2, 1) for t in (k, v))
        p = torch.softmax((q[s:e].double()[:, None] * kk[None]).sum(-1) * 0.2, 1)
        assert (got[s:e].double() - (p[..., None] * vv[None]).sum(1)).abs().max() < 2e-3


TILES = [  # Hq, Hk, D, P, lens, rows: prompt chunks, alone and beside others
    (4, 2, 64, 16, [1000], [1000]),
    (4, 1, 128, 64, [129], [65]),
    (8, 2, 128, 16, [700, 33, 1, 400, 90], [300, 1, 1, 64, 17]),
    (6, 1, 256, 128, [513, 77], [512, 30]),
    (9, 3, 64, 32, [5000, 64, 65], [150, 64, 65]),
    (2, 2, 128, 64, [3000, 300, 20, 2], [33, 300, 16, 2]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", TILES, ids=str)
def test_prompt_chunks(dev, shape, dtype, bits, causal):
    Hq, Hk, D, P, lens, rows = shape
    run(dev, dtype, bits, Hq, Hk, D, P, lens, rows, causal=causal, behind=3, max_rows=max(rows))


@pytest.mark.parametrize("bits", [16, 8])
def test_chunks_of_many_sequences(dev, bits):
    """More sequences than a wave has lanes; more items than workgroups run together; long ones split beside short ones."""
    run(dev, "bf16", bits, 2, 1, 64, 16, [40 + i % 90 for i in range(140)], [1 + (i * 7) % 40 for i in range(140)], max_rows=40)
    run(dev, "bf16", bits, 8, 8, 64, 16, [1200, 900], [1100, 800], max_rows=1100)
    run(dev, "f16", bits, 4, 2, 64, 64, [9000, 200, 100, 4000], [40, 200, 100, 33], max_rows=200)


@pytest.mark.parametrize("bits", [16, 8])
def test_chunk_rows_that_see_nothing(dev, bits):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(12)
    D, P, pool, T = 64, 16, 9, 150
    q = torch.randn(T, 4, D, generator=g).to(torch.bfloat16).to(dev)
    for table, starts, lens in (([[0, 1, 2, 3, 4]], [0, 120], [60]), ([[0, 1, -3, 3, 40, 5, 6, 7]], [0, 100], [120]), ([[0, 1, 2]], [3, 150], [999]),
                                ([[1, 2, 3, 4], [5, 6, 7, 8]], [0, 60, 90], [64, 64]), ([[1, 2], [5, 6]], [0, 160, 10], [32, 32]),
                                ([[-1] * 8], [0, 100], [128])):
        kp, vp = (make_pages(g, pool, 2, P, D, torch.bfloat16, bits, dev) for _ in range(2))
        args = (q, kp, vp, ints(table, dev), ints(starts, dev), ints(lens, dev))
        for causal in (True, False):
            got = ops.paged_attention(*args, scale=0.2, causal=causal)
            check(args, got, 0.2, causal)
            out = torch.full_like(q, 7.0)
            ops.paged_attention(*args, scale=0.2, causal=causal, out=out)
            none = np.isnan(attention(host(q), oracle_pages(kp), oracle_pages(vp), np.array(table), starts, lens, 0.2, causal)[0])
            none = torch.from_numpy(none).to(dev)
            assert (out[none] == 7).all() and torch.equal(out[~none], got[~none])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("split", [False, True])
def test_chunk_values_that_are_not_finite(dev, dtype, bits, split):
    """Behind the end and in keys that a row does not see they leave it alone; where it sees them they count."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(13)
    n, L = 80, 3000 if split else 200
    q, kp, vp, table, starts, lens = make(g, dev, dtype, bits, 4, 2, 64, 16, [L, 17], [n, 1])
    clean = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
    data = lambda p: p[0] if bits == 8 else p
    as_bits = lambda t: t.view(torch.uint8) if bits == 8 else t.view(torch.int16)
    bad = torch.full(data(kp).shape, float("nan"), device=dev).to(data(kp).dtype)
    used = torch.zeros(bad.shape[0], 16, dtype=torch.bool)
    for b, m in enumerate((L, 17)):
        for i in range(m):
            used[table[b, i // 16].item(), i % 16] = True
    for p in (kp, vp):
        as_bits(data(p)).copy_(torch.where((~used).to(dev)[:, None, :, None], as_bits(bad), as_bits(data(p))))
    assert torch.equal(ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125), clean)
    at = L - 10                                         # seen by the last ten rows
    for p in (kp, vp):
        keep = data(p).clone()
        as_bits(data(p))[table[0, at // 16].item(), :, at % 16] = as_bits(bad)[0, 0, 0, 0]
        got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
        assert not got[n - 10:n].isfinite().any() and got[:n - 10].isfinite().all() and torch.equal(got[n:], clean[n:])
        assert (got[:n - 10].double() - clean[:n - 10].double()).abs().max() <= 2 ** -7 * clean.double().abs().max()
        data(p).copy_(keep)
    if bits == 16:
        vp[table[0, 1].item(), :, 3, 5] = float("inf")
        got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125)
        assert (got[:n, :, 5] == float("inf")).all() and got[:n, :, :5].isfinite().all() and got[:n, :, 6:].isfinite().all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_chunk_scores_that_rise_and_fall(dev, dtype):
    """Scores that rise by little and by much from tile to tile, fall, and stand far under the first; values near the end of
    the type's range."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(14)
    q, kp, vp, table, starts, lens = make(g, dev, dtype, 16, 2, 1, 64, 16, [900], [70])
    q[:] = q[:1, :1]
    args = (q, kp, vp, table, starts, lens)
    for f in (lambda i: 0.001 * i, lambda i: 0.1 * i, lambda i: -0.1 * i, lambda i: 30.0 * (i == 0), lambda i: 3.0 * (i // 64 % 2), lambda i: -60 + 0.0 * i):
        for i in range(900):
            kp[table[0, i // 16].item(), :, i % 16] = q[0, 0] * (f(i) / 8)
        check(args, ops.paged_attention(*args, scale=0.125), 0.125)
    kp.zero_()
    vp.fill_(torch.finfo(DT[dtype]).max * 0.9)
    got = ops.paged_attention(*args, scale=0.125)
    assert torch.allclose(got.double(), vp[0, 0, 0, 0].double().expand(got.shape), rtol=2 ** -7, atol=0)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_chunks(dev, bits):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(15)
    q, kp, vp, table, _, _ = make(g, dev, "bf16", bits, 8, 2, 128, 16, [2000, 800, 40], [100, 3, 2])
    starts, lens = ints([0, 80, 83, 84], dev), ints([1500, 700, 3], dev)
    call = lambda: ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        lens += 7
        starts[1:] += 3
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check((q, kp, vp, table, starts, lens), out, 0.1)


def test_chunks_over_pages_of_extreme_scales(dev):
    """8-bit pages whose values do not fit fp16: the largest and the smallest scales, alone and beside ordinary ones."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(16)
    for low, high in ((-60, -59), (20, 21), (-30, 5)):
        q, kp, vp, table, starts, lens = make(g, dev, "bf16", 8, 4, 2, 64, 16, [400, 90], [100, 90])
        some = torch.randint(low, high, vp[1].shape, generator=g)
        some[torch.rand(vp[1].shape, generator=g) < 0.5] = low
        vp = (vp[0], (some + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(dev))
        args = (q, kp, vp, table, starts, lens)
        check(args, ops.paged_attention(*args, scale=0.125), 0.125)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D,Hq,Hk", [(128, 8, 2), (256, 6, 1), (64, 4, 4)])
def test_chunks_beside_decoded_tokens(dev, D, Hq, Hk, bits):
    """One launch or two, by pages and head dim: tokens and short blocks behind short and long caches beside a chunk, long ones
    split, sequences past the 64th among the split ones, rows of no sequence between and behind."""
    n = 70
    lens = [(53 * i) % 300 + 1 for i in range(n)]
    rows = [1 if i % 9 else 0 for i in range(n)]
    for i, L, r in ((3, 5000, 1), (40, 900, 250), (65, 7000, 2), (67, 3000, 33), (69, 4100, 16)):
        lens[i], rows[i] = L, r
    args, got = run(dev, "bf16", bits, Hq, Hk, D, 32, lens, rows, behind=5, max_rows=250, max_len=7000)
    q, kp, vp, table, starts, lens = args
    moved = starts.clone()
    moved[66:] += 3                             # three rows more for 65
    moved[65] -= 1                              # and one that was 64's
    args = q, kp, vp, table, moved, lens
    from dspark_rocm import ops

    check(args, ops.paged_attention(*args, scale=0.1, max_rows=250), 0.1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,lens", [([18, 40, 96, 3, 33, 64], [1500, 4007, 2900, 700, 64, 1111]), ([50], [6000]),
                                       ([11] * 64, [64 * i + 11 for i in range(64)]), ([11] * 66, [70 * i + 11 for i in range(66)])])
def test_verify_blocks_at_head_dim_256(dev, rows, lens, dtype):
    """Parts that all run together, where 64 sequences or fewer allow it."""
    run(dev, dtype, 16, 6, 1, 256, 32, [max(a, b) for a, b in zip(lens, rows)], rows, max_rows=max(rows))


def test_starts_that_fall(dev):
    """Starts whose differences pass 31 bits, and sequences that share rows, leave no row of a new output unwritten."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(21)
    kp, vp = (make_pages(g, 4, 1, 16, 64, torch.bfloat16, 16, dev) for _ in range(2))
    junk = [torch.full((1 << 16,), float("nan"), device=dev) for _ in range(4)]
    del junk                                    # what a new tensor finds in memory
    for T in (9, 200):
        q = torch.randn(T, 2, 64, generator=g).to(torch.bfloat16).to(dev)
        table = ints([[0, 1, 2, 3]] * 3, dev)
        for starts in ([0, 2 ** 31 - 1, -2, T], [0, T + 1, 0, T - 1], [0, 0, 0, 0], [T, T, T, T], [0, -2 ** 31, 2 ** 31 - 1, T]):
            args = q, kp, vp, table, ints(starts, dev), ints([30, 40, 50], dev)
            check(args, ops.paged_attention(*args, scale=0.2), 0.2)


def test_two_streams_at_once(dev):
    """Calls that overlap read the same pages, each with a workspace of its own."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(22)
    many = make(g, dev, "bf16", 16, 8, 2, 128, 64, [3000, 700], [200, 60])
    few = make(g, dev, "bf16", 16, 8, 2, 128, 64, [5000, 64, 1200], [1, 1, 4])
    want = [ops.paged_attention(*a, scale=0.1, max_rows=m) for a, m in ((many, 200), (few, 4))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, a, m in zip(streams, (many, few), (200, 4)):
            with torch.cuda.stream(s):
                got.append([ops.paged_attention(*a, scale=0.1, max_rows=m) for _ in range(4)])
        for s in streams:
            s.synchronize()
        assert all(torch.equal(x, w) for xs, w in zip(got, want) for x in xs)
