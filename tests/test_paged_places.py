"""CPU: what the paged-cache operators make of pools and tables without positions. The launches are left out."""

from __future__ import annotations

import pytest
import torch

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
