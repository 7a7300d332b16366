"""Tokens at the ends of the positions' range: what has no place is left out, and its
query is rotated unless its position is below 0 or past the rotation's tables."""
from __future__ import annotations

import pytest

from tests.test_paged import make, rand, rotate, tables

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
END = 2 ** 63 - 1


@gpu
@pytest.mark.parametrize("n_rot,neox", [(0, False), (0, True), (64, False), (64, True), (20, True)])
@pytest.mark.parametrize("start", [0, 5])
def test_ends_of_positions(n_rot, neox, start):
    n_kv, n_head, hd, n_pos = 2, 4, 64, 40
    c = make(n_kv, hd, 32, "f16", 3)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    at = [END, END - 1, n_pos, n_pos - 1, start + 3, 63 + start, 64 + start, 2 ** 32, -1, -2, -END,
          -END - 1, 2 ** 62]
    pos = torch.tensor(at, device="cuda")
    N = len(at)
    seq = torch.zeros_like(pos)
    q, k, v = rand(N, n_head * hd, seed=1), rand(N, n_kv * hd, seed=2), rand(N, n_kv * hd, seed=3)
    q_out = torch.full_like(q, 7.0)
    kw = {}
    if n_rot:
        kw = dict(zip(("cos", "sin"), tables(n_pos, n_rot)), neox=neox)
    c.append(k, v, table, pos, seq=seq, start=start, q=q, q_out=q_out, **kw)
    inside = torch.tensor([p >= 0 and (not n_rot or p < n_pos) for p in at], device="cuda")
    placed = inside & torch.tensor([start <= p < start + 64 for p in at], device="cuda")
    cos, sin = tables(n_pos, n_rot)
    turned = rotate(q.view(N, -1, hd), pos.clamp(0, n_pos - 1), cos, sin, neox).view(N, -1)
    assert torch.equal(q_out, torch.where(inside[:, None], turned, torch.full_like(q, 7.0)))
    gk, gv = c.read(table, pos, seq=seq, start=start)
    assert torch.equal(gv, torch.where(placed[:, None], v.half(), torch.zeros_like(gv)))
    assert int((c.v != 0).sum()) == int(placed.sum()) * n_kv * hd
    turned = rotate(k.view(N, -1, hd), pos.clamp(0, n_pos - 1), cos, sin, neox).view(N, -1)
    assert torch.equal(gk, torch.where(placed[:, None], turned.half(), torch.zeros_like(gk)))
