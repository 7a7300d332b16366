"""Attention over the paged cache with queries, keys and values of any size that bf16
and float32 hold.  Tolerance: that of tests/test_paged.py, whose check_attend this uses
(where scores are so large that their own rounding decides, it says no more than that
the output is a number)."""
from __future__ import annotations

import math

import pytest

from tests.test_paged import check_attend, rand, setting

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def scores(q, K, KP, n, n_kv, hd):
    """The largest |q.k| / sqrt(hd) of a row over its n positions, in 64 bits."""
    K = torch.cat([KP, K])[:n].double().permute(1, 0, 2).contiguous()
    qh = q.double().view(n_kv, -1, hd).permute(0, 2, 1).contiguous()
    return float(torch.bmm(K, qh).abs().max()) / math.sqrt(hd)


@gpu
@pytest.mark.parametrize("qscale,kscale", [
    (1.0, 1e30), (1.0, 1e35), (1.0, 5e37), (1e-10, 1e36), (1e-20, 1e20), (1e-30, 1e30),
    (1e-35, 1e35), (1e-37, 1e37), (3e-39, 3e37), (1e-18, 1e18), (1e-24, 1e24), (1e20, 1e-20),
    (1e35, 1e-35), (2e-20, 1.0)])
@pytest.mark.parametrize("n_head,n_kv,hd,N,own", [(8, 2, 64, 5, 50), (16, 2, 128, 40, 40),
                                                  (4, 2, 256, 3, 33)])
def test_bf16_keys_of_any_size(n_head, n_kv, hd, N, own, qscale, kscale):
    """Large keys of ordinary and of very small queries, down to subnormal ones, and
    small keys of large queries; rows of a common prefix in tiles of one row and more."""
    start = 130
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, "bf16", N, own, start,
                                             kscale=kscale)
    assert bool(K.isfinite().all()) and bool(KP.isfinite().all())
    q = (rand(N, n_head * hd, seed=14).double() * qscale).float()
    pos = (start + torch.arange(N) * 7 % own).cuda()
    pos[2] = 17
    # Scores above 2.3e38 are outside what the attention takes: in units of base 2 they
    # pass float32's range, 2^128 / log2(e) = 2.36e38.  (At 5e37 row 27 of the 40 has one
    # of 1.011 x 2^128 in these units, row 12 one of 1.000.)
    largest = [scores(q[i], K[i], KP, int(pos[i]) + 1, n_kv, hd) for i in range(N)]
    ok = torch.tensor([i for i in range(N) if largest[i] < 2.3e38], device="cuda")
    assert ok.numel() >= N - 2
    out = check_attend(c, q[ok], table, pos[ok], ok, K, V, prefix, start, KP, VP)
    assert bool(out.isfinite().all())


@gpu
def test_rows_of_different_sizes_together():
    """A tile's rows go by their own size each."""
    n_head, n_kv, hd, own, N = 8, 2, 64, 60, 20
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, "bf16", N, own, 64)
    scale = torch.tensor([1e-38, 1e-25, 1e-19, 6e-20, 1e-3, 1.0, 30.0, 0.0, 1e10, 1e-30] * 2)
    q = rand(N, n_head * hd, seed=21) * scale.cuda()[:, None]
    q[13, :64] *= 1e-20
    pos = (64 + torch.arange(N) * 3).cuda()
    want = check_attend(c, q, table, pos, None, K, V, prefix, 64, KP, VP)
    # a row's bits do not depend on its neighbours'
    alone = c.attend(q[5:6].expand(N, -1).contiguous(), table, pos, start=64, prefix=prefix)
    assert torch.equal(alone[5], want[5])


@gpu
@pytest.mark.parametrize("vscale", [1e-30, 1e10, 1e32, 1e35, 1e36])
@pytest.mark.parametrize("n_head,n_kv,hd,N,own,start", [
    (8, 2, 64, 5, 50, 130), (16, 2, 128, 40, 40, 64), (4, 2, 256, 3, 33, 30),
    (8, 1, 64, 2, 300, 0)])
def test_bf16_values_of_any_size(n_head, n_kv, hd, N, own, start, vscale):
    """Values whose weighted sums float32 holds (at most 300 of 4e36 each here)."""
    from tests.test_paged import fill
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, "bf16", N, own, start)
    V, VP = ((x.double() * vscale).bfloat16() for x in (V, VP))
    fill(c, table, K, V, start)
    if start:
        fill(c, prefix[None, :], KP[None], VP[None])
    q = rand(N, n_head * hd, seed=15)
    pos = (start + torch.arange(N) * 7 % own).cuda()
    pos[0] = start + own - 1
    out = check_attend(c, q, table, pos, None, K, V, prefix if start else None, start, KP, VP)
    assert bool(out.isfinite().all())


@gpu
def test_one_value_next_to_the_largest():
    """A row of one position gives its value, whatever it is."""
    c, table, prefix, K, V, KP, VP = setting(8, 2, 64, 32, "bf16", 3, 1, 0)
    top = torch.finfo(torch.bfloat16).max
    v = torch.linspace(-top, top, 3 * 2 * 64, dtype=torch.float64).bfloat16().view(3, 128).cuda()
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    c.append(rand(3, 128, seed=1), v.float(), table, pos)
    out = c.attend(rand(3, 512, seed=2), table, pos).view(3, 2, 4, 64)
    want = v.double().view(3, 2, 1, 64).expand(-1, -1, 4, -1)
    assert bool(((out.double() - want).abs() <= 2.0 ** -20 * want.abs()).all())
