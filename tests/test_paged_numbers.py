"""PagedKVCache: sizes past the C ABI's integers are refused, not taken by their low
bits."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kw", [dict(page_size=2 ** 32 + 64), dict(n_kv=2 ** 32 + 2),
                                dict(head_dim=2 ** 32 + 64), dict(n_pages=2 ** 64 + 4),
                                dict(n_kv=-2 ** 32 + 2), dict(n_pages=2 ** 31), dict(n_pages=0)])
def test_shapes(kw):
    from alpacca_amd.kvcache import PagedKVCache
    with pytest.raises(ValueError):
        PagedKVCache(**{**dict(n_kv=2, n_pages=4, head_dim=64, page_size=32), **kw})


@pytest.mark.gpu
def test_start():
    from alpacca_amd.kvcache import PagedKVCache
    c = PagedKVCache(2, 4, 64, page_size=32)
    table, pos = (torch.zeros(1, n, dtype=t, device="cuda") for n, t in (
        (4, torch.int32), (1, torch.int64)))
    k, pre = torch.ones(1, 128, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for start in (2 ** 64, 2 ** 63, -2 ** 64, -1):
        for call in (lambda: c.append(k, k, table, pos[0], start=start),
                     lambda: c.attend(k, table, pos[0], start=start, prefix=pre),
                     lambda: c.read(table, pos[0], start=start)):
            with pytest.raises(ValueError):
                call()
    assert not bool(c.k.any())
