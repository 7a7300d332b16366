"""The paged 16-bit KV cache (alpacca_amd.kvcache.PagedKVCache): what is stored
equals the rotation in fp32 rounded once, bit for bit; attention against the
softmax in 64 bits over the stored values; absent places, garbage behind the last
position, shared pages; refusals.

Tolerance of attention, per output component, from the arithmetic.  With
q in two (fp16) or three (bf16) pieces of at least 22 bits and fp32 accumulation, a
score z = q.k / sqrt(hd) is off by at most e_z = (hd 2^-24 + 2^-21) sum|q_d k_d| /
sqrt(hd) + 2^-23 |z| (sums, pieces, scale), which moves a weight by the factor
e^(2 e_z), the largest and its own; exponential, weights' pieces and the sum add
2^-20, and sums of n weighted values n_eff 2^-24 with n_eff below 64 + n / 32 (a
lane's own, then a tree).  All of it is times the weighted mean of |v|."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from alpacca_amd import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


def tables(n, n_rot, device="cuda"):
    inv = 10000.0 ** (-2.0 * torch.arange(n_rot // 2, dtype=torch.float64) / max(n_rot, 1))
    th = torch.arange(n, dtype=torch.float64)[:, None] * inv[None, :]
    return th.cos().float().contiguous().to(device), th.sin().float().contiguous().to(device)


def rotate(x, pos, cos, sin, neox):
    """x (N, heads, hd), each product and difference rounded to fp32."""
    half = cos.shape[1]
    if half == 0:
        return x
    cs, sn = cos[pos][:, None, :], sin[pos][:, None, :]
    a, b = ((slice(0, half), slice(half, 2 * half)) if neox
            else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    y, x0, x1 = x.clone(), x[..., a], x[..., b]
    p, r = x0 * cs, x1 * sn
    y[..., a] = p - r
    p, r = x0 * sn, x1 * cs
    y[..., b] = p + r
    return y


def make(n_kv, hd, page, dtype, n_pages):
    from alpacca_amd.kvcache import PagedKVCache
    return PagedKVCache(n_kv, n_pages, hd, page_size=page, dtype=DT[dtype])


def ids_of(n_pages, seed):
    return torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).int().cuda()


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


# ---- append and read ---------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd,n_rot,neox", [
    (8, 2, 64, 64, False), (8, 8, 64, 32, True), (14, 2, 128, 128, True), (5, 5, 128, 60, False),
    (32, 8, 128, 128, False), (4, 1, 256, 256, True), (16, 1, 256, 0, False), (6, 3, 64, 20, True),
    (2, 1, 64, 2, True)])
def test_append(n_head, n_kv, hd, n_rot, neox, dtype):
    page, seqs, width, start = 32, 5, 3, 37
    cos, sin = tables(200, n_rot)
    for N in (1, 7, 61):
        c = make(n_kv, hd, page, dtype, seqs * width + 4)
        table = ids_of(seqs * width + 4, N)[:seqs * width].view(seqs, width)
        slot = torch.randperm(seqs * width * page, generator=torch.Generator().manual_seed(N))[:N]
        seq, pos = (slot // (width * page)).cuda(), (slot % (width * page) + start).cuda()
        q, k, v = (rand(N, h * hd, seed=i + N) for i, h in ((1, n_head), (2, n_kv), (3, n_kv)))
        kw = dict(cos=cos, sin=sin, neox=neox) if n_rot else {}
        qr = c.append(k, v, table, pos, seq=seq, start=start, q=q, **kw)
        want_q = rotate(q.view(N, -1, hd), pos, cos, sin, neox).view(N, -1)
        want_k = rotate(k.view(N, -1, hd), pos, cos, sin, neox).view(N, -1).to(DT[dtype])
        assert torch.equal(qr, want_q)
        gk, gv = c.read(table, pos, seq=seq, start=start)
        assert torch.equal(gk, want_k) and torch.equal(gv, v.to(DT[dtype]))
        # nothing else was touched: as many values as were stored
        assert int((c.k != 0).sum()) <= k.numel() and int((c.v != 0).sum()) <= v.numel()
        # in place, without queries, and a prompt of one sequence in one call
        q2 = q.clone()
        assert c.append(k, v, table, pos, seq=seq, start=start, q=q2, q_out=q2, **kw) is q2
        assert torch.equal(q2, want_q)
        assert c.append(k, v, table, pos, seq=seq, start=start, **kw) is None
        assert torch.equal(c.read(table, pos, seq=seq, start=start)[0], want_k)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd,T", [(64, 1), (64, 200), (128, 31), (128, 97), (256, 65)])
def test_append_prompt(hd, T, dtype):
    """Runs of positions of one sequence, whole blocks and parts of them."""
    n_kv, page = 3, 64
    cos, sin = tables(1000, hd)
    for first in (0, 13, 32, 100):
        c = make(n_kv, hd, page, dtype, 9)
        table = ids_of(9, first)[None, :]
        k, v = rand(T, n_kv * hd, seed=first), rand(T, n_kv * hd, seed=first + 1)
        pos = torch.arange(first, first + T, device="cuda")
        c.append(k, v, table, pos, seq=torch.zeros_like(pos), cos=cos, sin=sin)
        every = torch.arange(9 * page, device="cuda")
        gk, gv = c.read(table, every, seq=torch.zeros_like(every))
        wk, wv = torch.zeros_like(gk), torch.zeros_like(gv)
        wk[first:first + T] = rotate(k.view(T, -1, hd), pos, cos, sin, False).view(T, -1).to(DT[dtype])
        wv[first:first + T] = v.to(DT[dtype])
        assert torch.equal(gk, wk) and torch.equal(gv, wv)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rounding_and_range(dtype):
    """Ties to even, subnormals, past the type's range, infinities and NaNs."""
    hd, dt = 64, DT[dtype]
    g = torch.Generator().manual_seed(1)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (6, 2 * hd), generator=g).to(torch.int32)
    x = bits.view(torch.float32).clone()
    half = (torch.arange(hd * 2).float() * 2 + 1) * (2.0 ** -25 if dtype == "f16" else 2.0 ** -9)
    x[1] = 1 + half % 1
    x[2] = torch.ldexp(torch.arange(2 * hd).float() + 0.5, torch.tensor(-24))
    x[3, :6] = torch.tensor([65504., 65519.9, 65520., -65520., INF, -INF])
    x[4] = torch.ldexp(torch.arange(2 * hd).float(), torch.tensor(-133))
    x = x.cuda()
    c = make(2, hd, 32, dtype, 1)
    pos = torch.arange(6, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    c.append(x, x.flip(0).contiguous(), table, pos, seq=torch.zeros_like(pos))
    k, v = c.read(table, pos, seq=torch.zeros_like(pos))
    for got, want in ((k, x.to(dt)), (v, x.flip(0).to(dt))):
        assert torch.equal(got.isnan(), want.isnan())
        ok = ~want.isnan()
        assert torch.equal(got.view(torch.int16)[ok], want.view(torch.int16)[ok])


@gpu
def test_tokens_without_a_place():
    n_kv, hd, page, n_head = 2, 64, 32, 4
    cos, sin = tables(90, hd)
    c = make(n_kv, hd, page, "f16", 6)
    table = torch.tensor([[0, 5, 99], [-1, 2, 3]], dtype=torch.int32, device="cuda")
    start = 10
    # (seq, pos): placed are only tokens 0, 3 and 8
    tok = [(0, 10), (0, 9), (0, -1), (1, 10 + 32), (2, 10), (-1, 10), (1, 10), (0, 10 + 64),
           (0, 41), (1, 10 + 96), (0, -2 ** 62), (0, 2 ** 62), (1, 89), (1, 90)]
    seq, pos = (torch.tensor(x, device="cuda") for x in zip(*tok))
    N = len(tok)
    q, k, v = rand(N, n_head * hd, seed=1), rand(N, n_kv * hd, seed=2), rand(N, n_kv * hd, seed=3)
    q_out = torch.full_like(q, 7.0)
    c.append(k, v, table, pos, seq=seq, start=start, cos=cos, sin=sin, q=q, q_out=q_out)
    placed = torch.tensor([i in (0, 3, 8, 12) for i in range(N)], device="cuda")
    gk, gv = c.read(table, pos, seq=seq, start=start)
    assert torch.equal(gv, torch.where(placed[:, None], v.half(), torch.zeros_like(gv)))
    assert int((c.v != 0).sum()) == 4 * n_kv * hd
    inside = (pos >= 0) & (pos < 90)
    want = rotate(q.view(N, -1, hd), pos.clamp(0, 89), cos, sin, False).view(N, -1)
    assert torch.equal(q_out, torch.where(inside[:, None], want, torch.full_like(q, 7.0)))
    # seq None: row i is token i's; more tokens than rows
    c2 = make(n_kv, hd, page, "f16", 6)
    c2.append(k[:4], v[:4], table, torch.tensor([0, 40, 3, 3], device="cuda"))
    assert int((c2.v != 0).sum()) == 2 * n_kv * hd
    # a table without pages, and no tokens
    c2.append(k[:4], v[:4], table[:, :0], pos[:4], seq=seq[:4])
    c2.append(k[:0], v[:0], table, pos[:0])
    assert c2.read(table, pos[:0])[0].shape == (0, n_kv * hd)
    assert int((c2.v != 0).sum()) == 2 * n_kv * hd


# ---- attention ---------------------------------------------------------------------

def attend64(q, K, V, hd, n_kv):
    """q (n_head * hd) over K, V (n, n_kv, hd), all float64: the output and the
    tolerance of the module's comment, both (n_head, hd)."""
    n = K.shape[0]
    G = q.numel() // (n_kv * hd)
    qh = q.view(n_kv, G, hd)
    if n == 0:
        z = torch.zeros(n_kv * G, hd, dtype=torch.float64, device=q.device)
        return z, z
    Kt = K.permute(1, 2, 0).contiguous()
    z = torch.bmm(qh, Kt) / math.sqrt(hd)
    mag = torch.bmm(qh.abs(), Kt.abs()) / math.sqrt(hd)
    p = torch.softmax(z, dim=2)
    Vh = V.permute(1, 0, 2).contiguous()
    out, vabs = torch.bmm(p, Vh), torch.bmm(p, Vh.abs())
    # the errors of the scores that carry the weight, at their largest
    big = p > 2.0 ** -30
    ez = ((hd * 2.0 ** -24 + 2.0 ** -21) * mag + 2.0 ** -23 * z.abs()) * big
    ez = ez.amax(2, keepdim=True)
    tol = (torch.expm1(2 * ez) + 2.0 ** -20 + (64 + n / 32) * 2.0 ** -24) * vabs + 2.0 ** -29 * \
        Vh.abs().amax(1, keepdim=True)
    return out.view(-1, hd), tol.view(-1, hd)


def fill(c, table, K, V, start=0):
    """K, V (seqs, n, n_kv, hd) into the rows of the table."""
    seqs, n = K.shape[:2]
    pos = torch.arange(start, start + n, device="cuda").repeat(seqs)
    seq = torch.arange(seqs, device="cuda").repeat_interleave(n)
    c.append(K.reshape(seqs * n, -1).float(), V.reshape(seqs * n, -1).float(), table, pos, seq=seq,
             start=start)


def check_attend(c, q, table, pos, seq, K, V, prefix=None, start=0, KP=None, VP=None, **kw):
    """K, V (seqs, slots, n_kv, hd), KP, VP (start, n_kv, hd): what the pages hold."""
    out = c.attend(q, table, pos, seq=seq, start=start, prefix=prefix, **kw)
    hd, n_kv = c.head_dim, c.n_kv
    for i in range(q.shape[0]):
        b, p = (i if seq is None else int(seq[i])), int(pos[i])
        own = max(0, min(p + 1 - start, K.shape[1])) if p >= 0 and 0 <= b < K.shape[0] else 0
        parts = [(K[b, :own], V[b, :own])] if own else []
        if start and p >= 0:
            parts.insert(0, (KP[:min(start, p + 1)], VP[:min(start, p + 1)]))
        Ki = torch.cat([x[0] for x in parts]).double() if parts else K[0, :0].double()
        Vi = torch.cat([x[1] for x in parts]).double() if parts else V[0, :0].double()
        want, tol = attend64(q[i].double(), Ki, Vi, hd, n_kv)
        err = (out[i].view(-1, hd).double() - want).abs()
        assert bool((err <= tol).all()), (i, b, p, float((err - tol).max()), float(err.max()))
    return out


def setting(n_head, n_kv, hd, page, dtype, seqs, own, start, seed=0, kscale=1.0, spare=0):
    width, n_pre = -(-own // page), -(-start // page)
    total = seqs * width + n_pre + spare
    c = make(n_kv, hd, page, dtype, max(total, 1))
    ids = ids_of(total, seed)
    prefix, table = ids[:n_pre], ids[n_pre:n_pre + seqs * width].view(seqs, width)
    K, V = (rand(seqs, own, n_kv, hd, seed=seed + i) for i in (1, 2))
    KP, VP = (rand(start, n_kv, hd, seed=seed + i) for i in (3, 4))
    K, KP = K * kscale, KP * kscale
    K, V, KP, VP = (x.to(DT[dtype]) for x in (K, V, KP, VP))
    if own:
        fill(c, table, K, V, start)
    if start:
        fill(c, prefix[None, :], KP[None], VP[None])
    return c, table, prefix, K, V, KP, VP


HEADS = [(8, 2, 64), (8, 8, 64), (14, 2, 128), (32, 8, 128), (16, 1, 64), (5, 1, 256), (12, 4, 256),
         (3, 3, 128), (33, 3, 64)]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd", HEADS)
def test_attend_own(n_head, n_kv, hd, dtype):
    """Each row over its own pages: lengths from none to several pages."""
    page, own = 32, 230
    pos = [0, 1, 30, 31, 32, 33, 63, 64, 100, 229, -1, 128]
    c, table, _, K, V, _, _ = setting(n_head, n_kv, hd, page, dtype, len(pos), own, 0, seed=hd)
    q = rand(len(pos), n_head * hd, seed=9)
    check_attend(c, q, table, torch.tensor(pos, device="cuda"), None, K, V)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd", HEADS)
@pytest.mark.parametrize("start", [1, 64, 523])
def test_attend_prefix(n_head, n_kv, hd, dtype, start):
    page, own, seqs = 64, 90, 6
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, page, dtype, seqs, own, start,
                                             seed=start)
    pos = torch.tensor([start + x for x in (0, 5, 31, 32, 80, 89)], device="cuda")
    q = rand(seqs, n_head * hd, seed=10)
    check_attend(c, q, table, pos, None, K, V, prefix, start, KP, VP)
    # rows that end inside the prefix, padding, rows without a row of the table
    pos = torch.tensor([0, start - 1, start // 2, -1, start + 89, start], device="cuda")
    seq = torch.tensor([0, 1, 2, 3, 7, -1], device="cuda")
    check_attend(c, q, table, pos, seq, K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd,N,start,own", [
    (32, 8, 128, 64, 2051, 40), (32, 8, 64, 70, 999, 300), (16, 2, 128, 33, 4097, 65),
    (4, 4, 64, 257, 700, 33), (16, 1, 256, 40, 600, 33), (8, 1, 256, 19, 3001, 10),
    (28, 4, 128, 40, 300, 70), (2, 1, 64, 500, 260, 5)])
def test_attend_many_rows(n_head, n_kv, hd, N, start, own, dtype):
    """Enough rows that the prefix's products are shared by tiles of rows."""
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, dtype, N, own, start, seed=N)
    g = torch.Generator().manual_seed(N)
    pos = (start + torch.randint(0, own, (N,), generator=g)).cuda()
    pos[3] = start // 3
    pos[5] = -1
    q = rand(N, n_head * hd, seed=11)
    check_attend(c, q, table, pos, None, K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("n_head,n_kv,hd,T", [(8, 2, 64, 5), (14, 2, 128, 4), (4, 1, 256, 3)])
def test_attend_several_tokens(n_head, n_kv, hd, T):
    """Tokens of one sequence checked together, each over those before it."""
    page, own, seqs, start = 64, 200, 3, 70
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, page, "f16", seqs, own, start)
    first = torch.tensor([0, 61, 190])
    pos = (start + first[:, None] + torch.arange(T)[None, :]).reshape(-1).cuda()
    seq = torch.arange(seqs).repeat_interleave(T).cuda()
    q = rand(seqs * T, n_head * hd, seed=12)
    check_attend(c, q, table, pos, seq, K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 64), (14, 2, 128), (3, 3, 128), (8, 1, 256),
                                            (10, 1, 64)])
@pytest.mark.parametrize("start", [0, 70])
def test_attend_runs_of_tokens(n_head, n_kv, hd, start):
    """Tokens of one sequence beside one another in every manner: runs longer than
    a tile and across 64 tokens, positions in any order and the same twice, padding
    and rows that end inside the prefix between them, rows out of the table."""
    seqs, own = 4, 150
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, "f16", seqs, own, start, seed=hd)
    g = torch.Generator().manual_seed(n_head + start)
    N = 150
    seq = torch.randint(0, seqs, (N,), generator=g).sort().values
    seq[60:70] = seq[64]  # a run across the border
    seq[:70:7] = 3
    seq[100], seq[101], seq[102] = 9, 9, -1
    pos = start + torch.randint(0, own, (N,), generator=g)
    pos[30:40] = torch.arange(start + 20, start + 30)
    pos[41:44] = start + 77
    pos[50] = -1
    pos[52] = max(start - 3, 0)
    q = rand(N, n_head * hd, seed=18)
    check_attend(c, q, table, pos.cuda(), seq.cuda(), K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("start", [0, 64])
def test_positions_past_the_table(start):
    """A row attends to all that its row of the table holds, alone or in a run."""
    seqs, own, end = 3, 96, (1 << 63) - 1
    c, table, prefix, K, V, KP, VP = setting(8, 2, 64, 32, "f16", seqs, own, start, seed=7)
    pos = torch.tensor([start + 4, end, start + 95, start + 96, end - 1, end, start], device="cuda")
    q = rand(7, 8 * 64, seed=20)
    for seq in ([0, 0, 0, 1, 1, 1, 2], [0, 1, 2, 0, 1, 2, 0], [2] * 7):
        check_attend(c, q, table, pos, torch.tensor(seq, device="cuda"), K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd,T", [(8, 2, 64, 4), (14, 2, 128, 2), (4, 4, 128, 16)])
def test_tokens_do_not_see_what_comes_after_them(n_head, n_kv, hd, T, dtype):
    """Infinities and NaNs at a position reach the tokens of its sequence that attend
    to it, and not those beside them that end before it, in the same block or an
    earlier one."""
    own, seqs = 100, 2
    c, table, _, K, V, _, _ = setting(n_head, n_kv, hd, 32, dtype, seqs, own, 0)
    pos = torch.tensor([(90 - 5 * t) % 97 for t in range(T)]).repeat(seqs).cuda()
    seq = torch.arange(seqs).repeat_interleave(T).cuda()
    q = rand(seqs * T, n_head * hd, seed=19)
    want = check_attend(c, q, table, pos, seq, K, V)
    for value in (float("nan"), INF, -INF):
        at = torch.tensor([88], device="cuda")
        x = torch.full((1, n_kv * hd), value, device="cuda")
        c.append(x, x, table[1:], at, seq=torch.zeros_like(at))
        got = c.attend(q, table, pos, seq=seq)
        hit = (seq == 1) & (pos >= 88)
        assert bool(hit.any()) and torch.equal(got[~hit], want[~hit])
        assert bool((~got[hit].isfinite()).any(1).all())


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_long(dtype):
    """Long own pages of few rows, and a long prefix of one row."""
    for n_head, n_kv, hd, seqs, own, start in ((8, 2, 128, 2, 9001, 0), (8, 1, 64, 1, 33, 20011),
                                               (4, 2, 256, 1, 4100, 3000)):
        c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 128, dtype, seqs, own, start)
        pos = torch.tensor([start + own - 1, start + own // 2][:seqs], device="cuda")
        q = rand(seqs, n_head * hd, seed=13)
        check_attend(c, q, table, pos, None, K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("qscale,kscale", [(1e-30, 1.0), (30.0, 1.0), (1.0, 1e-4), (300.0, 30.0),
                                           (1e30, 1e-4), (0.0, 1.0)])
def test_attend_scales(dtype, qscale, kscale):
    """Scores from next to nothing to far past exp's range; subnormal keys."""
    n_head, n_kv, hd, start, own = 8, 2, 64, 130, 50
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, dtype, 5, own, start,
                                             kscale=kscale)
    q = rand(5, n_head * hd, seed=14) * qscale
    pos = torch.tensor([start, start + 3, start + 20, start + 49, 17], device="cuda")
    check_attend(c, q, table, pos, None, K, V, prefix, start, KP, VP)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("N", [4, 70])
def test_garbage_behind_the_last_position(dtype, N):
    """What lies behind a row's last position, in its page and in later ones, or
    in pages that no row names, is never used, whatever it is; a row of NaN
    queries does not reach the others."""
    n_head, n_kv, hd, start, own = 16, 4, 64, 45, 96
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, dtype, N, own, start, spare=3)
    every = torch.arange(c.n_pages, device="cuda").int()
    used = torch.cat([table.flatten(), prefix])
    bad = torch.tensor([float("nan"), INF, -INF, 65000.0], device="cuda").repeat(n_kv * hd // 4)
    # unused pages; slots behind the prefix's last; slots behind each row's last
    rest = every[~torch.isin(every, used)][None, :]
    pos = (start + torch.arange(N) * 7 % own).cuda()
    spots = [(rest, torch.arange(rest.shape[1] * 32, device="cuda"), 0, None),
             (prefix[None, :], torch.arange(start, 64, device="cuda"), 0, None)]
    for b in range(N):
        spots.append((table[b:b + 1], torch.arange(int(pos[b]) + 1, start + own, device="cuda"),
                      start, None))
    for tab, p, st, _ in spots:
        if p.numel():
            x = bad.repeat(p.numel(), 1)
            c.append(x, x, tab, p, seq=torch.zeros_like(p), start=st)
    q = rand(N, n_head * hd, seed=15)
    out = check_attend(c, q, table, pos, None, K, V, prefix, start, KP, VP)
    q2 = q.clone()
    q2[1] = float("nan")
    out2 = c.attend(q2, table, pos, start=start, prefix=prefix)
    keep = torch.arange(N, device="cuda") != 1
    assert torch.equal(out2[keep], out[keep]) and bool(out2[1].isnan().all())
    # an infinity or a NaN among the values attended to shows in those rows alone
    at = torch.tensor([start], device="cuda")
    c.append(bad[None, :], bad[None, :], table[2:3], at, seq=torch.zeros_like(at), start=start)
    out3 = c.attend(q, table, pos, start=start, prefix=prefix)
    keep = torch.arange(N, device="cuda") != 2
    assert torch.equal(out3[keep], out[keep]) and bool(out3[2].isnan().any())


@gpu
def test_pages_out_of_range_and_shared_pages():
    """Page numbers outside the pool leave their positions out; rows may share
    pages of their own."""
    n_head, n_kv, hd, page, own, start = 8, 2, 64, 32, 160, 96
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, page, "f16", 4, own, start)
    q = rand(4, n_head * hd, seed=16)
    pos = torch.tensor([start + 159, start + 70, start + 33, start + 10], device="cuda")
    t2, p2 = table.clone(), prefix.clone()
    t2[0, 1], t2[1, 0], t2[2], t2[3] = -1, 2 ** 31 - 1, c.n_pages, -2 ** 31
    p2[1] = -5
    out = c.attend(q, t2, pos, start=start, prefix=p2)
    for i in range(4):
        own_at = [s for s in range(int(pos[i]) - start + 1)
                  if 0 <= int(t2[i, s // page]) < c.n_pages]
        pre_at = [s for s in range(start) if s // page != 1]
        Ki = torch.cat([KP[pre_at], K[i, own_at]]).double()
        Vi = torch.cat([VP[pre_at], V[i, own_at]]).double()
        want, tol = attend64(q[i].double(), Ki, Vi, hd, n_kv)
        assert bool(((out[i].view(-1, hd).double() - want).abs() <= tol).all())
    # nothing at all to attend to
    nothing = torch.full_like(table, -1)
    assert not bool(c.attend(q, nothing, pos, start=0).any())
    assert not bool(c.attend(q, table[:, :0], pos, start=0).any())
    assert not bool(c.attend(q, table[:0], pos, start=0).any())
    # all rows read row 1's pages
    same = table[1:2].expand(4, -1)
    a = c.attend(q, same, pos, start=start, prefix=prefix)
    b = c.attend(q, table, pos, seq=torch.ones(4, dtype=torch.int64, device="cuda"), start=start,
                 prefix=prefix)
    assert torch.equal(a, b)


@gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^31 values: places near its end."""
    n_kv, hd, page = 8, 256, 128
    n_pages = 2 ** 31 // (n_kv * hd * page) + 40
    c = make(n_kv, hd, page, "bf16", n_pages)
    assert c.k.numel() > 2 ** 31
    table = torch.tensor([[n_pages - 1, 3, n_pages - 7], [0, n_pages - 2, 5]], dtype=torch.int32,
                         device="cuda")
    K, V = rand(2, 384, n_kv, hd, seed=1).bfloat16(), rand(2, 384, n_kv, hd, seed=2).bfloat16()
    fill(c, table, K, V)
    pos = torch.tensor([383, 200], device="cuda")
    gk, gv = c.read(table, pos)
    assert torch.equal(gk, torch.stack([K[0, 383], K[1, 200]]).view(2, -1))
    assert torch.equal(gv, torch.stack([V[0, 383], V[1, 200]]).view(2, -1))
    check_attend(c, rand(2, 16 * hd, seed=3), table, pos, None, K, V)


@gpu
def test_views_out_and_repeatability():
    """Strided and unaligned inputs, rows in three dimensions, out, the same bits
    from run to run and on another stream."""
    n_head, n_kv, hd, start, own, N = 8, 2, 64, 300, 70, 9
    c, table, prefix, K, V, KP, VP = setting(n_head, n_kv, hd, 32, "f16", N, own, start)
    q = rand(N, n_head * hd, seed=17)
    pos = (start + torch.arange(N) * 7).cuda()
    want = c.attend(q, table, pos, start=start, prefix=prefix)
    wide = torch.zeros(N, 2 * n_head * hd + 1, device="cuda")
    wide[:, 1::2] = q
    flat = torch.zeros(q.numel() + 1, device="cuda")
    flat[1:] = q.flatten()
    out = torch.full_like(q, 3.0)
    for x, kw in ((wide[:, 1::2], {}), (flat[1:].view(N, -1), {}), (q, dict(out=out)),
                  (q.view(N, n_head, hd), {})):
        got = c.attend(x, table, pos, start=start, prefix=prefix, **kw)
        assert torch.equal(got.reshape(N, -1), want) and got.shape == x.shape
    t2 = torch.zeros(N, 2 * table.shape[1], dtype=torch.int32, device="cuda")
    t2[:, ::2] = table
    p2 = torch.zeros(2 * N, dtype=torch.int64, device="cuda")
    p2[::2] = pos
    assert torch.equal(c.attend(q, t2[:, ::2], p2[::2], start=start, prefix=prefix), want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = c.attend(q, table, pos, start=start, prefix=prefix)
    s.synchronize()
    assert torch.equal(got, want)
    # the bits of a row do not depend on the other rows' values
    q3 = q * 2
    q3[4] = q[4]
    assert torch.equal(c.attend(q3, table, pos, start=start, prefix=prefix)[4], want[4])


@gpu
def test_decode_loop_with_sampling_captured():
    """The operators together as a decode step uses them: logits to a token, its
    keys and values (rows of an embedding) appended, attention over prefix and own
    pages; captured, replayed with eager work between, and equal to the eager loop."""
    from alpacca_amd.logits import sample_logits, sampling_params
    n_head, n_kv, hd, page, start, N, n_vocab, steps = 8, 2, 64, 32, 75, 6, 500, 40
    g = torch.Generator().manual_seed(0)
    emb, wk, wv, wo = (torch.randn(*s, generator=g).cuda() * f for s, f in (
        ((n_vocab, n_head * hd), 1.0), ((n_head * hd, n_kv * hd), 0.05),
        ((n_head * hd, n_kv * hd), 0.05), ((n_head * hd, n_vocab), 0.1)))
    cos, sin = tables(400, hd)
    par = sampling_params(None, 0.9, 40, 0.95, 0.01)
    U = torch.rand(steps, N, generator=g, dtype=torch.float64).cuda()
    width = -(-(steps + 1) // page)
    n_pre = -(-start // page)
    ids = ids_of(n_pre + N * width, 3)
    prefix, table = ids[:n_pre], ids[n_pre:].view(N, width)
    KP, VP = rand(start, n_kv * hd, seed=20), rand(start, n_kv * hd, seed=21)

    def fresh():
        c = make(n_kv, hd, page, "f16", n_pre + N * width)
        at = torch.arange(start, device="cuda")
        c.append(KP, VP, prefix[None, :], at, seq=torch.zeros_like(at), cos=cos, sin=sin)
        return c, torch.arange(N, device="cuda"), torch.full((N,), start, device="cuda")

    def step(c, tok, pos, u):
        x = emb[tok]
        q = c.append(x @ wk, x @ wv, table, pos, start=start, cos=cos, sin=sin, q=x)
        logits = c.attend(q, table, pos, start=start, prefix=prefix) @ wo
        sample_logits(logits, u, par, out=tok)
        pos += 1
        return logits

    c, tok, pos = fresh()
    want = []
    for i in range(steps):
        step(c, tok, pos, U[i])
        want.append(tok.clone())
    assert len(torch.stack(want).unique()) > 20
    c, tok, pos = fresh()
    u = U[0].clone()
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step(c, tok.clone(), pos.clone(), u)  # (the products' workspaces)
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        step(c, tok, pos, u)
    for i in range(steps):
        with torch.cuda.stream(s):
            u.copy_(U[i])
            graph.replay()
        s.synchronize()
        assert torch.equal(tok, want[i]), i
        c.attend(rand(N, n_head * hd, seed=i), table, pos, start=start, prefix=prefix)  # eager
        torch.cuda.synchronize()


# ---- refusals ----------------------------------------------------------------------

def test_shapes_refused():
    lib = _lib.load()
    size = ctypes.c_size_t()

    def sizes(n_kv=8, n_pages=10, hd=128, page=64, dtype=1):
        c = _lib.Paged(None, None, n_pages, page, n_kv, hd, dtype)
        return lib.aq_paged_sizes(ctypes.addressof(c), ctypes.byref(size))
    assert sizes() == _lib.AQ_OK and size.value == 10 * 64 * 8 * 128 * 2
    for kw in (dict(n_kv=0), dict(n_pages=0), dict(n_pages=2 ** 31), dict(hd=96), dict(hd=512),
               dict(page=16), dict(page=0), dict(page=48), dict(page=-32), dict(page=2 ** 17),
               dict(dtype=0), dict(dtype=8), dict(n_kv=65536),
               dict(n_pages=2 ** 31 - 1, page=65536)):
        assert sizes(**kw) == _lib.AQ_ERR_VALUE, kw
    assert lib.aq_paged_sizes(None, ctypes.byref(size)) == _lib.AQ_ERR_VALUE


def test_c_arguments_refused():
    lib, p, odd = _lib.load(), 4096, 4100
    good = dict(k=p, v=p, n_pages=4, page_size=32, n_kv=2, head_dim=64, dtype=1)

    def cache(**kw):
        return _lib.Paged(*[dict(good, **kw)[f] for f, _ in _lib.Paged._fields_])

    def append(c=None, q=p, k=p, v=p, qo=p, N=1, n_head=4, n_rot=64, cos=p, sin=p, n_pos=9, table=p,
               seqs=1, width=1, pos=p, start=0):
        c = cache() if c is None else c
        return lib.aq_rope_paged(q, k, v, qo, N, n_head, n_rot, 0, cos, sin, n_pos, table, seqs,
                                 width, None, pos, start, ctypes.addressof(c), None)

    def attend(c=None, q=p, N=1, n_head=4, table=p, seqs=1, width=1, pos=p, prefix=p, n_prefix=1,
               start=0, scratch=p, size=1 << 40, out=p):
        c = cache() if c is None else c
        return lib.aq_attention_paged(q, ctypes.addressof(c), N, n_head, table, seqs, width, None,
                                      pos, prefix, n_prefix, start, scratch, size, out, None)

    def read(c=None, N=1, table=p, seqs=1, width=1, pos=p, start=0, k=p, v=p):
        c = cache() if c is None else c
        return lib.aq_paged_read(ctypes.addressof(c), N, table, seqs, width, None, pos, start, k,
                                 v, None)
    bad = _lib.AQ_ERR_VALUE
    for fn in (append, attend, read):
        for c in (cache(k=None), cache(v=None), cache(k=odd), cache(v=odd), cache(head_dim=80),
                  cache(page_size=8)):
            assert fn(c=c) == bad
        for kw in (dict(N=-1), dict(N=2 ** 24 + 1), dict(seqs=-1), dict(width=-1), dict(start=-1),
                   dict(seqs=2 ** 31), dict(width=2 ** 31), dict(pos=None), dict(table=None)):
            assert fn(**kw) == bad, (fn, kw)
        assert fn(N=0) == _lib.AQ_OK
    for kw in (dict(k=None), dict(v=None), dict(qo=None), dict(n_rot=66), dict(n_rot=3),
               dict(n_rot=-2), dict(cos=None), dict(sin=None), dict(n_pos=-1), dict(n_head=0),
               dict(q=odd), dict(k=odd), dict(v=odd), dict(qo=odd)):
        assert append(**kw) == bad, kw
    for kw in (dict(q=None), dict(out=None), dict(q=odd), dict(out=odd), dict(n_head=3),
               dict(n_head=34), dict(n_head=0), dict(n_prefix=-1), dict(start=33),
               dict(start=1, n_prefix=0), dict(start=1, prefix=None), dict(N=2 ** 23)):
        assert attend(**kw) == bad, kw
    for kw in (dict(k=None), dict(v=None), dict(k=odd), dict(v=odd)):
        assert read(**kw) == bad, kw


@gpu
def test_python_arguments_refused():
    from alpacca_amd.kvcache import PagedKVCache
    for kw in (dict(head_dim=80), dict(page_size=40), dict(dtype=torch.float32), dict(n_pages=0),
               dict(device="cpu")):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_kv=2, n_pages=4, head_dim=64), **kw})
    c = PagedKVCache(2, 4, 64, page_size=32)
    assert c.dtype == torch.float16 and c.storage_nbytes() == 4 * 32 * 2 * 64 * 4
    N = 3
    table, pos = torch.arange(3, device="cuda").int().view(3, 1), torch.zeros(
        N, dtype=torch.int64, device="cuda")
    k, q = torch.zeros(N, 128, device="cuda"), torch.zeros(N, 256, device="cuda")
    cos, sin = tables(4, 64)
    ok = dict(k=k, v=k, table=table, pos=pos, cos=cos, sin=sin, q=q)
    c.append(**ok)
    for kw in (dict(k=k[:2]), dict(v=k[:2]), dict(k=k.half()), dict(q=q[:2]), dict(q=k[:, :64]),
               dict(pos=pos[:2]), dict(pos=pos.int()), dict(table=table[0]), dict(start=-1),
               dict(table=table.long()), dict(table=table.cpu()), dict(seq=pos[:2]),
               dict(seq=pos.int()), dict(cos=cos[:2]), dict(cos=cos.double()), dict(sin=None),
               dict(q_out=q[:2]), dict(q=None, q_out=q), dict(k=k.cpu()),
               dict(cos=torch.zeros(4, 40, device="cuda"), sin=torch.zeros(4, 40, device="cuda"))):
        with pytest.raises(ValueError):
            c.append(**{**ok, **kw})
    ok = dict(q=q, table=table, pos=pos)
    c.attend(**ok)
    pre = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in (dict(q=q[:2]), dict(q=q[:, :100]), dict(start=1), dict(start=33, prefix=pre),
               dict(start=1, prefix=pre.long()), dict(start=1, prefix=pre[None]), dict(start=-1),
               dict(out=q[:2]), dict(out=q.half()), dict(q=torch.zeros(3, 34 * 64, device="cuda"))):
        with pytest.raises(ValueError):
            c.attend(**{**ok, **kw})
    assert c.attend(q[:0], table, pos[:0]).shape == (0, 256)
