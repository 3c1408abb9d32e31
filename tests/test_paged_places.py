"""CPU: what the paged-cache operators make of pools and tables without positions. The launches are left out."""

from __future__ import annotations

import pytest
import torch

from dspark_rocm import ops
from tests.test_paged_inputs import BF, append, attend, case, host, pages  # noqa: F401 (host: a fixture)


@pytest.mark.parametrize("codes", [False, True])
def test_pools_and_tables_of_nothing(host, codes):
    """Rows of sequences still are turned, and see nothing: the kernels are called with a table that leads nowhere."""
    d = case(codes)
    cut = lambda p: tuple(t[:0] for t in p) if codes else p[:0]
    for kw in (dict(table=d["table"][:, :0]), dict(table=d["table"][:, :0].long()), dict(k_pages=cut(d["k_pages"]), v_pages=cut(d["v_pages"]))):
        c = {**d, **kw, "q_out": torch.ones(3, 4, 64, dtype=BF)}
        assert append(c) is c["q_out"]
        name, f = host.pop()
        assert name == "dspark_paged_append" and f[2:7] == (4, 2, 64, 16, 1)
        assert f[-4:] == (1, 2, 1, 3)
        out = torch.ones(3, 4, 64, dtype=BF)
        c = {n: t for n, t in c.items() if n != "q_out"}
        assert attend(c, out=out, workspace=torch.zeros(8, dtype=torch.uint8)) is out
        name, f = host.pop()
        assert name == "dspark_paged_attention" and f[6] == 1 and f[-6:-2] == (1, 2, 1, 3) and f[-1] >= 256
    with pytest.raises(ValueError, match="no heads"):
        append(case(k=d["k"][:, :0], v=d["v"][:, :0], k_pages=pages()[:, :0], v_pages=pages()[:, :0]))
    assert not host


def shifted(buf, at, shape, stride):
    return buf.as_strided(shape, stride, at)


def test_appends_that_write_what_they_read_or_write(host):
    """Shifted views of one buffer, pages inside a pool, pools that run into each other: refused, whatever their first addresses."""
    buf = torch.zeros(4, 2, 64, dtype=BF)
    pool = torch.zeros(8, 2, 16, 64, dtype=BF)
    d = case(q=torch.zeros(3, 2, 64, dtype=BF))
    inside = pool[1, :, :3].transpose(0, 1)
    codes, scales = torch.zeros(8, 2, 16, 64).to(torch.float8_e4m3fn), torch.zeros(8, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    p8, raw = pages(True), torch.zeros(768, dtype=torch.uint8)
    for kw in (dict(q_out=buf[:3], k=buf[1:]), dict(q_out=buf[1:], v=buf[:3]), dict(q_out=inside, k_pages=pool[:5]), dict(q_out=inside, v_pages=pool[:5]),
               dict(k_pages=pool[:5], v_pages=pool[3:]), dict(k_pages=pool[1:6], v_pages=pool[:5]),
               dict(k_pages=(codes[:5], p8[1]), v_pages=(codes[3:], pages(True)[1])), dict(k_pages=(codes[:5], scales[:5]), v_pages=(p8[0], scales[1:6])),
               dict(k_pages=shifted(pool, 0, (5, 2, 16, 64), (3072, 1024, 64, 1)), v_pages=shifted(pool, 1024, (5, 2, 16, 64), (3072, 1024, 64, 1))),
               dict(k_pages=p8, v_pages=(pages(True)[0], raw[256:266].view(5, 2).view(torch.float8_e8m0fnu)), q_out=raw.view(BF).view(3, 2, 64))):
        with pytest.raises(ValueError, match="twice"):
            append({**d, **kw})
    with pytest.raises(ValueError, match="overlaps the pages"):
        attend(case(), q=d["q"], k_pages=pool[:5], v_pages=pool[:5], out=inside)
    with pytest.raises(ValueError, match="overlaps the pages"):
        attend(case(), q=d["q"], v_pages=pool[2:7], k_pages=pages(), out=pool[6, :, 13:].transpose(0, 1))
    assert not host


def test_appends_to_interleaved_views(host):
    """One buffer's heads, one pool's halves, by page, by head and by position; the queries in place; pages read from one pool by
    attention while their neighbours are written."""
    x = torch.zeros(3, 8 * 64, dtype=BF)
    q, k, v = (t.unflatten(1, (-1, 64)) for t in x.split([256, 128, 128], 1))
    append(case(q=q, k=k, v=v, q_out=q))
    append(case(q=torch.zeros(3, 4, 64, dtype=BF), k=k, v=v, q_out=q))
    y = torch.zeros(3, 2, 3, 64, dtype=BF)                   # each KV head's query, key and value
    append(case(q=y[:, :, 0], k=y[:, :, 1], v=y[:, :, 2], q_out=y[:, :, 0]))
    for shape, dim in (((2, 5, 2, 16, 64), 0), ((5, 2, 2, 16, 64), 1), ((5, 2, 2, 16, 64), 2), ((5, 2, 16, 2, 64), 3), ((5, 2, 16, 128), 3)):
        both = torch.zeros(shape, dtype=BF)
        append(case(k_pages=both.select(dim, 0) if len(shape) == 5 else both[..., :64], v_pages=both.select(dim, 1) if len(shape) == 5 else both[..., 64:]))
        codes = both.to(torch.float8_e4m3fn)
        scales = torch.zeros(5, 2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        halves = (codes.select(dim, 0), codes.select(dim, 1)) if len(shape) == 5 else (codes[..., :64], codes[..., 64:])
        append(case(k_pages=(halves[0], scales[..., 0]), v_pages=(halves[1], scales[..., 1])))
    pool = torch.zeros(10, 2, 16, 64, dtype=BF)
    append(case(k_pages=pool[::2], v_pages=pool[1::2]))
    append(case(k_pages=pool[:5], v_pages=pool[5:], k=pool[3, :, :3].transpose(0, 1), v=pool[8, :, 2:5].transpose(0, 1)))
    wide = torch.zeros(5, 2, 16, 192, dtype=BF)              # a pool beside rows that others use
    attend(case(), k_pages=wide[..., :64], v_pages=wide[..., 64:128], q=torch.zeros(3, 2, 64, dtype=BF), out=wide[:3, :, 0, 128:])
    assert len(host) == 16


def test_views_apart_or_not_by_counting():
    """What is said to lie apart shares no byte, counted one by one; the usual interleaved layouts are found."""
    import itertools
    import random

    rng = random.Random(1)
    said = 0
    for _ in range(3000):
        a, b = (tuple((rng.randint(1, 4), rng.choice((0, 1, 2, 3, 4, 6, 8, 12, 16, 24))) for _ in range(rng.randint(1, 3))) for _ in range(2))
        ahead, size = rng.randint(-30, 30), rng.choice((1, 2))
        cells = lambda at, dims: {at + sum(i * s for i, (_, s) in zip(at_, dims)) + e for at_ in itertools.product(*(range(n) for n, _ in dims)) for e in range(size)}
        apart = not cells(0, a) & cells(ahead, b)
        got = ops._lie_apart(ahead, size, a, size, b)
        assert apart or not got
        assert ops._share(ops._span(100, size, *a), ops._span(100 + ahead, size, *b)) or apart
        said += got
    assert said > 200
