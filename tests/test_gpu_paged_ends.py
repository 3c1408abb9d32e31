"""GPU: paged caches at the ends of their ranges: keys and scales that a narrower type does not hold, scores and scales without a
number, chunks that begin again."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_ref
from tests._paged import DT, attention, check_rows, exps, host, ints, make_pages, make_table, oracle_pages, starts_of, typed

pytestmark = pytest.mark.gpu

BEHIND = {1: 40, 5: 3000, 100: 150, 33: 6000}          # rows: positions; one part and several, of either kernel


def call(args, scale, pieces=2.0 ** -16, **kw):
    """The operator's rows, against attention in 64 bits over the values that the pages hold."""
    from dspark_rocm import ops

    q, kp, vp, table, starts, lens = args
    got = ops.paged_attention(*args, scale=scale, **kw)
    want, tol = attention(host(q), oracle_pages(kp), oracle_pages(vp), table.cpu().numpy(), starts.tolist(), lens.tolist(), scale, True, pieces)
    check_rows(got, want, tol)
    return got


def make(g, dev, dtype, bits, Hq, Hk, D, P, lens, rows):
    pool = sum(-(-n // P) for n in lens) + 2
    kp, vp = (make_pages(g, pool, Hk, P, D, DT[dtype], bits, dev) for _ in range(2))
    q = torch.randn(sum(rows), Hq, D, generator=g).to(DT[dtype]).to(dev)
    return q, kp, vp, make_table(g, lens, P, pool, dev), starts_of(rows, dev), ints(lens, dev)


def with_scales(pages, e):
    return pages[0], (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(pages[0].device)


# ---------------------------------------------------------------------------- 8-bit keys that fp16 does not hold


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", BEHIND)
def test_the_largest_keys_of_fp16_rows(dev, n, D, both):
    """A row's 65000 becomes the code 256 of scale 2^8: 65536, which fp16 does not have and a score does. Keys of one sign, and of
    both; queries of either."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(1)
    L = BEHIND[n]
    q, kp, vp, table, starts, lens = make(g, dev, "f16", 8, 2, 1, D, 16, [L], [n])
    k, v = (torch.randn(L, 1, D, generator=g).to(torch.float16) for _ in range(2))
    k[::3, 0, 5] = 65000.0
    if both:
        k[1::3, 0, 5] = -65504.0
    ops.paged_append(k.to(dev), v.to(dev), kp, vp, table, ints([0, L], dev), lens)
    assert (oracle_pages(kp).values == 65536).any()
    for far in (-1e-4, 1e-4, 3e-5):
        q[..., 5] = far
        call((q, kp, vp, table, starts, lens), 0.125)


def test_one_key_that_fp16_does_not_hold(dev):
    """The only key of a row has all of its weight, whatever its score."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(2)
    q, kp, vp, table, starts, lens = make(g, dev, "f16", 8, 1, 1, 64, 16, [1], [1])
    k, v = torch.full((1, 1, 64), 1.0, dtype=torch.float16, device=dev), torch.ones(1, 1, 64, dtype=torch.float16, device=dev)
    k[..., 0] = 65000.0
    ops.paged_append(k, v, kp, vp, table, starts, lens)
    q[..., 0] = -1e-4
    assert (ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.125) == 1).all()


@pytest.mark.parametrize("low,high,size", [(8, 14, 2e-5), (-26, -20, 3e4), (-24, 12, 1e-3)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", BEHIND)
def test_scales_of_keys_past_fp16(dev, n, D, low, high, size):
    """Scales past both ends of fp16, pages of ordinary ones between."""
    g = torch.Generator().manual_seed(3)
    q, kp, vp, table, starts, lens = make(g, dev, "f16", 8, 2, 1, D, 16, [BEHIND[n]], [n])
    e = torch.randint(low, high, kp[1].shape, generator=g)
    e[torch.rand(e.shape, generator=g) < 0.3] = -7
    q = (q * size).clamp(-65504, 65504)
    call((q, with_scales(kp, e), vp, table, starts, lens), 0.05)


# ---------------------------------------------------------------------------- rows without a finite score


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", BEHIND)
def test_rows_whose_scores_are_all_minus_infinity(dev, n, D, dtype):
    """exp(-inf - -inf) is no number: an infinity in every key that a row sees is not hidden behind a zero. Rows that see nothing
    of their sequence, or a finite score beside, are what they were."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(4)
    L = BEHIND[n]
    q, kp, vp, table, starts, lens = make(g, dev, dtype, 16, 2, 1, D, 16, [L, 90], [n, 1])
    q[:, 0, 3], q[:, 1, 3] = 1.0, 0.5
    clean = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    for b, m in enumerate((L, 90)):
        if b == 0:
            kp[table[b, :-(-m // 16)].long(), :, :, 3] = -float("inf")
    got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    assert got[:n].isnan().all() and torch.equal(got[n:], clean[n:])
    kp[table[0, 0].item(), :, 7, 3] = 2.0                    # one key that has a score
    got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    seen = torch.arange(L - n, L, device=dev) >= 7
    assert torch.equal(got[:n][seen], vp[table[0, 0].item(), :, 7].expand(int(seen.sum()), 2, D)) and got[:n][~seen].isnan().all()
    # of n rows the last 7 have positions: the others see nothing
    if n > 7:
        kp[table[0, 0].item(), :, 7, 3] = -float("inf")
        short = lens.clone()
        short[0] = 7
        got = ops.paged_attention(q, kp, vp, table, starts, short, scale=0.1)
        assert not got[:n - 7].any() and got[n - 7:n].isnan().all()
        gone = table.clone()
        gone[0] = -1
        assert not ops.paged_attention(q, kp, vp, gone, starts, lens, scale=0.1)[:n].any()


@pytest.mark.parametrize("n", BEHIND)
def test_scores_far_below_zero(dev, n):
    """Equal scores of -1e34, one product each: finite, and a softmax like that of zeros."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(5)
    L = BEHIND[n]
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 16, 2, 1, 64, 16, [L], [n])
    q.zero_()
    kp.zero_()
    q[..., 0], kp[..., 0] = 1e17, -1e17
    got = ops.paged_attention(q, kp, vp, table, starts, lens, scale=1.0)
    want, tol = attention(0 * host(q), oracle_pages(kp), oracle_pages(vp), table.cpu().numpy(), starts.tolist(), lens.tolist(), 1.0)
    check_rows(got, want, tol)


# ---------------------------------------------------------------------------- every scale byte


def values(pages):
    """What codes with scale bytes stand for, in 64 bits: 2^-127 for byte 0, NaN for 255."""
    b = pages[1].view(torch.uint8).cpu().numpy().astype(np.float64)
    return host(pages[0]) * np.where(b == 255, np.nan, np.exp2(b - 127))[:, :, None, None]


def with_bytes(pages, b):
    return pages[0], torch.as_tensor(b, dtype=torch.uint8).expand(pages[1].shape).contiguous().view(torch.float8_e8m0fnu).to(pages[0].device)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_read_of_every_scale_byte(dev, dtype):
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(6)
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1, 4).view(256, 1, 16, 64).view(torch.float8_e4m3fn).to(dev)
    pages = with_bytes((codes, torch.zeros(256, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)), torch.arange(256)[:, None])
    other = make_pages(g, 256, 1, 16, 64, DT[dtype], 8, dev)
    k, v = ops.paged_read(pages, other, torch.arange(256, dtype=torch.int32, device=dev), dtype=DT[dtype])
    for got, p in ((k, pages), (v, other)):
        np.testing.assert_array_equal(host(got), typed(DT[dtype])(values(p)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", BEHIND)
def test_attention_over_every_scale_byte(dev, n, dtype):
    """A NaN scale is NaN to the rows that see its page and nothing to others; the least and the largest are numbers."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(7)
    L = BEHIND[n]
    q, kp, vp, table, starts, lens = make(g, dev, dtype, 8, 2, 1, 64, 16, [L, 90], [n, 1])
    clean = ops.paged_attention(q, kp, vp, table, starts, lens, scale=0.1)
    last = table[0, (L - 1) // 16].item()
    sees = torch.arange(L - n, L, device=dev) >= (L - 1) // 16 * 16
    for which in (0, 1):
        pages = [kp, vp]
        b = pages[which][1].view(torch.uint8).clone()
        b[last] = 255
        pages[which] = with_bytes(pages[which], b)
        got = ops.paged_attention(q, *pages, table, starts, lens, scale=0.1)
        assert got[:n][sees].isnan().all() and torch.equal(got[n:], clean[n:])
        off = (got[:n][~sees].double() - clean[:n][~sees].double()).abs()
        assert off.numel() == 0 or off.max() <= 2 ** -7 * clean.double().abs().max()
    # keys and values of next to nothing, values that fp16 does not hold beside them (there: rows computed again in fp32)
    for which in (0, 1):
        pages = [kp, vp]
        b = pages[which][1].view(torch.uint8).clone()
        b[::2] = 0
        if which and dtype == "f16":
            b[1::2] = 127 + 8
        pages[which] = with_bytes(pages[which], b)
        x = host(q), *(paged_ref.Pages(values(p)) for p in pages)
        want, tol = attention(*x, table.cpu().numpy(), starts.tolist(), lens.tolist(), 0.1, True, 2.0 ** (-11 if dtype == "bf16" else -16))
        got = ops.paged_attention(q, *pages, table, starts, lens, scale=0.1)
        fits = np.abs(want) < 6e4
        check_rows(torch.where(torch.from_numpy(fits).to(dev), got, 0), np.where(fits, want, 0), tol)
        assert fits.mean() > 0.5


@pytest.mark.parametrize("which", [254, 255, 0])
def test_rows_behind_the_last_scales(dev, which):
    """A page's old scale counts where it holds rows before: 2^127 as any other, NaN for the new rows too."""
    from dspark_rocm import ops

    g = torch.Generator().manual_seed(8)
    D, P = 64, 16
    kp, vp = (with_bytes(make_pages(g, 2, 2, P, D, torch.bfloat16, 8, dev), torch.full((2, 2), which)) for _ in range(2))
    k, v = (torch.randn(3, 2, D, generator=g).to(torch.bfloat16) * (1e38 if which else 1.0) for _ in range(2))
    k, v = k.clamp(-3e38, 3e38), v.clamp(-3e38, 3e38)
    want = []
    for pages, x in ((kp, k), (vp, v)):
        w = paged_ref.Pages(values(pages), np.full((2, 2), which - 127))
        if which != 255:
            paged_ref.append(w, host(x), np.array([[1]]), [0, 3], [8])
        else:
            w.values[1, :, 5:8] = np.nan
        want.append(w)
    ops.paged_append(k.to(dev), v.to(dev), kp, vp, ints([[1]], dev), ints([0, 3], dev), ints([8], dev))
    for got, w in zip((kp, vp), want):
        np.testing.assert_array_equal(exps(got[1]), w.exps)
        np.testing.assert_array_equal(values(got)[:, :, :8], w.values[:, :, :8])


# ---------------------------------------------------------------------------- no positions at all


@pytest.mark.parametrize("bits", [16, 8])
def test_pools_and_tables_of_nothing(dev, bits):
    """A pool without pages, a table without room: rows of sequences are turned, and see nothing; rows of none stay."""
    from dspark_rocm import ops, rope

    g = torch.Generator().manual_seed(9)
    freqs = rope.frequencies(64, 1e4, device=dev)[0]
    q, kp, vp, table, _, _ = make(g, dev, "bf16", bits, 4, 2, 64, 16, [40, 3], [5, 2])
    starts, lens = ints([1, 4, 6], dev), ints([40, 3], dev)
    k, v = (torch.randn(7, 2, 64, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    cut = lambda p: tuple(t[:0] for t in p) if bits == 8 else p[:0]
    want = ops.paged_append(k, v, kp, vp, torch.full_like(table, -1), starts, lens, q=q, freqs=freqs)
    inside = torch.tensor([False] + [True] * 5 + [False], device=dev)
    for pages, t in (((kp, vp), table[:, :0]), ((cut(kp), cut(vp)), table), ((cut(kp), cut(vp)), table[:, :0].long())):
        assert torch.equal(ops.paged_append(k, v, *pages, t, starts, lens, q=q, freqs=freqs), want)
        y = q.clone()
        assert ops.paged_append(k, v, *pages, t, starts, lens, q=y, freqs=freqs, q_out=y) is y
        assert torch.equal(y[inside], want[inside]) and torch.equal(y[~inside], q[~inside])
        for rows in (1, 7):
            out = torch.full_like(q, 7.0)
            ops.paged_attention(q, *pages, t, starts, lens, scale=0.1, out=out, max_rows=rows)
            assert not out[inside].any() and (out[~inside] == 7).all()
            assert not ops.paged_attention(q, *pages, t, starts, lens, scale=0.1, max_rows=rows).any()
        assert ops.paged_append(k, v, *pages, t, starts, lens) is None
    assert not inside.all() and want[inside].any()


# ---------------------------------------------------------------------------- 8-bit chunks of bf16 models: one fp16 piece, or again with two


def chunk(args, scale, **kw):
    """A probability is one fp16 piece: half a step, 2^-11 of it at most, or where it is subnormal, 2^-25 with the row's reference at
    2^7: 2^-32 of the largest weight a key."""
    from dspark_rocm import ops

    q, kp, vp, table, starts, lens = args
    got = ops.paged_attention(*args, scale=scale, **kw)
    values = oracle_pages(vp)
    want, tol = attention(host(q), oracle_pages(kp), values, table.cpu().numpy(), starts.tolist(), lens.tolist(), scale, True, 2.0 ** -11)
    check_rows(got, want, tol + int(lens.max()) * 2.0 ** -32 * np.abs(values.values).max())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("low,high", [(-60, -59), (20, 21), (-30, 5), (-3, -1)])
def test_chunks_that_begin_again(dev, D, low, high):
    """V that does not fit fp16 in some page of every item, early or late."""
    g = torch.Generator().manual_seed(10)
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 8, 4, 2, D, 16, [700, 90, 2000], [200, 90, 33])
    e = torch.randint(low, high, vp[1].shape, generator=g)
    e[torch.rand(e.shape, generator=g) < 0.5] = low
    chunk((q, kp, with_scales(vp, e), table, starts, lens), 0.125)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("e", [-2, 12, -40, -110])
@pytest.mark.parametrize("rows,L,at", [(33, 6000, 5200), (33, 6000, 40), (600, 1500, 1390), (70, 9000, 4500)])
def test_one_page_that_does_not_fit(dev, D, e, rows, L, at):
    """One page among many: the part, or the row tiles, that come to it begin again, the others do not, and are joined."""
    g = torch.Generator().manual_seed(11)
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 8, 2, 1, D, 16, [L, 300], [rows, 40])
    b = (vp[1].view(torch.uint8).to(torch.int64) - 127).cpu()
    b[table[0, at // 16].item()] = e
    chunk((q, kp, with_scales(vp, b), table, starts, lens), 0.1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,L", [(100, 700), (33, 6000), (600, 1500)])
def test_chunks_with_pages_that_are_not_there(dev, D, rows, L):
    g = torch.Generator().manual_seed(12)
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 8, 2, 1, D, 16, [L, 300], [rows, 40])
    for at, bad in ((L // 2, -1), (L // 2 + 16, 10 ** 6), (L - 1, -7), (0, -1)):
        table[0, at // 16] = bad
        chunk((q, kp, vp, table, starts, lens), 0.1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,L", [(70, 900), (33, 6000)])
@pytest.mark.parametrize("shape", ["slow", "rise", "fall", "first", "steps", "low", "late"])
def test_8_bit_scores_that_rise_and_fall(dev, D, rows, L, shape):
    """The running maximum's rule where a probability is fp16: up to 2^8 over the reference, and far under it."""
    from dspark_rocm import ops

    f = {"slow": lambda i: 0.001 * i, "rise": lambda i: 0.02 * i, "fall": lambda i: -0.02 * i, "first": lambda i: 30.0 * (i == 0),
         "steps": lambda i: 5.4 * (i // 64 % 2), "low": lambda i: -60 + 0.0 * i, "late": lambda i: 25.0 * (i == L - rows)}[shape]
    g = torch.Generator().manual_seed(13)
    q, kp, vp, table, starts, lens = make(g, dev, "bf16", 8, 2, 1, D, 16, [L], [rows])
    q[:] = q[:1, :1]
    size = float((q[0, 0].double() ** 2).sum()) * 0.1
    k = (q[0, 0].double()[None, None] * f(torch.arange(L, dtype=torch.float64, device=dev))[:, None, None] / size).to(torch.bfloat16)
    v = torch.randn(L, 1, D, generator=g).to(torch.bfloat16).to(dev)
    ops.paged_append(k, v, kp, vp, table, ints([0, L], dev), lens)
    chunk((q, kp, vp, table, starts, lens), 0.1)


@pytest.mark.parametrize("Hq,Hk,D,P,lens,rows", [(4, 2, 64, 16, [1, 2, 5, 900], [1, 2, 4, 3]), (32, 8, 128, 64, [3, 700, 40], [2, 16, 1]),
                                                 (6, 1, 256, 32, [4, 1300, 2], [1, 5, 2]), (8, 1, 128, 16, [2500, 9], [8, 6])])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_few_rows_over_8_bit_pages_have_two_pieces(dev, Hq, Hk, D, P, lens, rows, dtype):
    """Decoded tokens and verify blocks: 2^-16 of a probability, over 8-bit pages too. Few keys, where a piece lost is not averaged
    away."""
    for seed in range(4):
        g = torch.Generator().manual_seed(20 + seed)
        call(make(g, dev, dtype, 8, Hq, Hk, D, P, lens, rows), D ** -0.5, max_rows=max(rows), max_len=max(lens))
