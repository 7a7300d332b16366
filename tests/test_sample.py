"""Sampling (aq_sample through alpacca_amd.logits): tokens equal to the definition
evaluated in 64 bits, log-probabilities to fp32's rounding; refusals (on the CPU).

Tolerances.  The kernel adds weights as whole multiples of 2^-e of the largest,
e = 62 - bits(n): a sum of n of them is off by n 2^-(e + 1) at most, plus a double
exponential's 2^-50 or so each.  Where u times the sum lies nearer to a border than
SLACK of the sum, the oracle takes either side's token; that happens to a row in
1e7 here.  So it does where top-p times the sum lies that near to one, for the same
reason: of 200 equal logits 0.9 keeps 180 if the product is rounded to a double, 181 if
it is not, as the double 0.9 is 0.9 + 2.2e-17, and so do other tokens whose weights are
2e-13 together.  A logarithm is rounded to fp32 once: 2^-24 of it, beside 1e-9 for the
sum."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from alpacca_amd import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
SLACK = 1e-9


def order_of(x):
    """Tokens above -inf, by logit descending, then by number."""
    x = np.where(np.isnan(x), -np.inf, x)
    t = np.flatnonzero(x > -np.inf)
    return t[np.lexsort((t, -x[t].astype(np.float64)))]


def kept_of(x, temp, k, p, min_p):
    """The order's kept beginning, its weights and how far they are weights."""
    o = order_of(x)
    if len(o) == 0 or not temp > 0:
        return o[:1], np.ones(len(o[:1]))
    v = x[o].astype(np.float64)
    with np.errstate(all="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / temp))
    keep = len(o)
    if k >= 1:
        keep = min(keep, int(min(k, 2 ** 31)))
    run = np.cumsum(w[:keep])
    if p < 1:
        keep = min(keep, int(np.searchsorted(run, p * run[-1], side="left")) + 1)
    if min_p > 0:
        keep = min(keep, max(1, int((w >= min_p).sum())))
    return o[:keep], w[:keep]


def want(x, u, temp, k, p, min_p):
    """The tokens that may come out, and their log-probabilities (for each way to take
    top-p's border)."""
    u = min(max(u if u == u else 0.0, 0.0), 1 - 2 ** -53)
    out = {}
    for share in sorted({p, p * (1 - SLACK), p * (1 + SLACK)} if p < 1 else {p}):
        o, w = kept_of(x, temp, k, share, min_p)
        if len(o) == 0:
            return {-1: {-np.inf}}
        run = np.cumsum(w)
        for g in (u - SLACK, u, u + SLACK):
            i = min(int(np.searchsorted(run, g * run[-1], side="right")), len(o) - 1)
            while i > 0 and w[i] == 0:
                i -= 1
            with np.errstate(divide="ignore"):
                lp = float(np.log(w[i]) - np.log(run[-1])) if temp > 0 else 0.0
            out.setdefault(int(o[i]), set()).add(lp)
    return out


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check(x, u, par):
    from alpacca_amd.logits import sample_logits
    x, u, par = np.asarray(x, np.float32), np.asarray(u, np.float64), np.asarray(par, np.float64)
    tok, lp = sample_logits(dev(x), dev(u), dev(par), logp=True)
    tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
    for r in range(len(x)):
        ok = want(x[r], float(u[r]), *(par[r] if par.ndim == 2 else par))
        assert int(tok[r]) in ok, (r, int(tok[r]), ok, u[r], par)
        refs = ok[int(tok[r])]
        assert any(lp[r] == ref if math.isinf(ref) else
                   abs(lp[r] - ref) <= abs(ref) * 2 ** -24 + 1e-9 + 1e-12 * abs(ref)
                   for ref in refs), (r, lp[r], refs)


def logits(rng, rows, n, spread=3.0):
    x = spread * rng.standard_normal((rows, n))
    m = min(n, 50)
    for r in range(rows):
        x[r, rng.choice(n, m, replace=False)] += 12 - rng.uniform(1, 3) * np.log(np.arange(1, m + 1))
    return x.astype(np.float32)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (0.7, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.02),
            (1.0, 1, 1.0, 0.0), (0.0, 5, 0.5, 0.5), (1.1, 300, 1.0, 0.0), (2.5, 0, 0.99, 0.0),
            (1.0, 0, 1e-9, 0.0), (1.0, 10 ** 9, 1.0, 1.0), (0.05, 0, 1.0, 0.0),
            (1.0, 7, 0.6, 0.3), (30.0, 5000, 0.8, 1e-4)]


@gpu
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 2), (5, 63), (3, 64), (3, 65), (4, 1000),
                                    (2, 2048), (1, 4097), (9, 32003), (2, 128256), (1, 262145)])
def test_settings(rows, n):
    rng = np.random.default_rng(rows * 7 + n)
    x = logits(rng, rows, n)
    for par in SETTINGS:
        u = rng.random(rows)
        check(x, u, par)


@gpu
def test_each_row_its_own():
    rng = np.random.default_rng(5)
    rows, n = 3 * len(SETTINGS), 20011
    check(logits(rng, rows, n), rng.random(rows), np.array(SETTINGS * 3))


@gpu
@pytest.mark.parametrize("n", [40003, 9001])
@pytest.mark.parametrize("m", [1, 63, 64, 65, 128, 129, 200, 256, 257, 511, 512, 513, 1024, 1025,
                               4095, 4096, 4097, 8000])
def test_lengths_of_what_is_kept(m, n):
    """As many tokens far above the others as each way of ordering takes, and one
    more: scattered, together at the row's end, and in groups of equal ones."""
    rng = np.random.default_rng(m)
    x = rng.standard_normal((6, n)).astype(np.float32) - 40
    head = (0.002 * np.arange(m)[::-1]).astype(np.float32)
    for r in range(6):
        where = rng.choice(n, m, replace=False) if r % 2 else np.arange(n - m, n)
        x[r, rng.permutation(where) if r < 4 else where] = head if r < 2 else np.floor(2 * head)
    for par in ((1.0, m, 1.0, 0.0), (1.0, m, 0.97, 0.0), (3.0, 0, 0.999, 0.0), (1.0, 0, 0.9, 1e-3)):
        check(x, rng.random(6), par)


@gpu
@pytest.mark.parametrize("heavy", [2, 3, 17, 64, 500])
def test_heavy_tokens_side_by_side(heavy):
    """What is kept lies together, where the largest of 64 tokens each say little of
    the sum; and a body that weighs little, as much, or most."""
    rng = np.random.default_rng(heavy)
    n, rows = 30011, 8
    x = rng.standard_normal((rows, n)).astype(np.float32)
    for r in range(rows):
        first = int(rng.integers(0, n - heavy)) if r % 2 else 640 + 64 * r
        x[r, first:first + heavy] = 8 + 0.7 * r - rng.uniform(0, 0.5, heavy)
    for par in ((0.9, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 0, 0.999, 1e-4), (0.8, 0, 0.5, 0.0),
                (1.0, heavy, 0.9, 0.0)):
        check(x, rng.random(rows), par)


@gpu
@pytest.mark.parametrize("u", [0.0, 1e-300, 0.25, 0.5, 1 - 2 ** -53, 1.0, 7.0, -3.0, np.nan])
def test_ends_of_u(u):
    rng = np.random.default_rng(11)
    x = logits(rng, 4, 5003)
    x[1] = 1.5  # all the same
    x[2] = -np.inf
    x[2, 77] = -3.0
    x[3, 10:] = -np.inf
    for par in SETTINGS:
        check(x, np.full(4, u), par)


@gpu
@pytest.mark.parametrize("n", [4, 4096, 4100, 100001])
def test_equal_logits(n):
    """More equal logits than are sorted at once, at the top and below it: the
    lowest tokens come first."""
    rng = np.random.default_rng(n)
    x = np.full((6, n), 0.25, np.float32)
    x[1, ::2] = -0.5
    x[2, 1::3] = 1.0
    x[3] = np.where(rng.random(n) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[4] = np.float32(2.0) + np.float32(2 ** -22) * rng.integers(0, 3, n)
    x[5, :2] = 9.0
    for par in SETTINGS + [(1.0, n // 2, 1.0, 0.0), (1.0, n // 2 + 1, 0.37, 0.0)]:
        for _ in range(2):
            check(x, rng.random(6), par)


@gpu
def test_values_at_the_ends():
    """Masked by -inf, by the lowest float, infinities, NaNs, subnormals, large
    magnitudes, rows that hold nothing."""
    rng = np.random.default_rng(3)
    n = 3001
    x = rng.standard_normal((9, n)).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0] = np.where(rng.random(n) < 0.99, -np.inf, x[0])
    x[1] = np.where(rng.random(n) < 0.99, low, x[1])
    x[2] = low
    x[3] = -np.inf
    x[4, [5, 9, 2000]] = np.inf
    x[5, ::7] = np.nan
    x[6] = np.nan
    x[7] = np.float32(1e-42) * rng.integers(0, 30, n)
    x[8] *= np.float32(1e37)
    for par in SETTINGS:
        check(x, rng.random(9), par)


@gpu
def test_odd_params():
    """NaN counts as left out, a negative number as 0; a fraction of top_k is
    dropped; extreme temperatures."""
    rng = np.random.default_rng(4)
    x = logits(rng, 2, 3000)
    u = rng.random(2)
    from alpacca_amd.logits import sample_logits
    nan = np.nan

    def tokens(par):
        return sample_logits(dev(x), dev(u), dev(np.array(par, np.float64))).cpu().tolist()
    assert tokens((1.0, nan, nan, nan)) == tokens((1.0, 0, 1, 0))
    assert tokens((1.0, -4, 2.0, -1.0)) == tokens((1.0, 0, 1, 0))
    assert tokens((1.0, 5.9, 1, 0)) == tokens((1.0, 5, 1, 0))
    first = x.argmax(1).tolist()
    for t in (nan, -1.0, 0.0, 1e-310, 1e-30):
        assert tokens((t, 0, 1, 0)) == first
    assert tokens((1.0, 0, -2.0, 0)) == first
    assert tokens((1.0, 0, 1, 9.0)) == first
    check(x, u, (1e30, 0, 1.0, 0.0))
    check(x, u, (np.inf, 0, 1.0, 0.0))


@gpu
def test_frequencies():
    """Over evenly spread u every token comes out as often as its share says, to
    the two draws that a border can move."""
    from alpacca_amd.logits import sample_logits
    rng = np.random.default_rng(6)
    n, m = 40, 4000
    x = (2 * rng.standard_normal(n)).astype(np.float32)
    u = (np.arange(m) + 0.5) / m
    par = (0.9, 20, 0.9, 0.01)
    tok = sample_logits(dev(np.tile(x, (m, 1))), dev(u), dev(np.array(par))).cpu().numpy()
    o, w = kept_of(x, *par)
    share = np.zeros(n)
    share[o] = w / w.sum()
    assert np.abs(np.bincount(tok, minlength=n) - m * share).max() <= 2


@gpu
def test_one_dimension_views_streams_and_capture():
    from alpacca_amd.logits import sample_logits, sampling_params
    rng = np.random.default_rng(8)
    n = 9001
    x = logits(rng, 3, n)
    par = sampling_params(None, 0.9, 50, 0.9, 0.01)
    assert par.shape == (4,) and sampling_params(3, 0.9, [1, 2, 3]).shape == (3, 4)
    u = rng.random(3)
    xd, ud = dev(x), dev(u)
    all_rows = sample_logits(xd, ud, par)
    for r in range(3):
        one = sample_logits(xd[r], ud[r], par)
        assert one.shape == () and int(one) == int(all_rows[r])
    wide = torch.zeros(3, 2 * n, device="cuda")
    wide[:, ::2] = xd
    assert torch.equal(sample_logits(wide[:, ::2], ud, par), all_rows)
    assert sample_logits(xd[:0], ud[:0], par).shape == (0,)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    out = torch.empty(3, dtype=torch.int64, device="cuda")
    with torch.cuda.graph(g, stream=s):
        sample_logits(xd, ud, par, out=out)
    for i in range(4):
        u = rng.random(3)
        with torch.cuda.stream(s):
            out.fill_(-7)
            ud.copy_(dev(u))
            g.replay()
        s.synchronize()
        eager = sample_logits(xd, dev(u), par)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals():
    from alpacca_amd.logits import sample_logits, sampling_params
    x, u, par = torch.zeros(2, 8), torch.zeros(2, dtype=torch.float64), sampling_params(
        None, device="cpu")
    with pytest.raises(ValueError, match="must be on a GPU"):
        sample_logits(x, u, par)
    with pytest.raises(ValueError, match="float32 tensor"):
        sample_logits(x.double(), u, par)
    with pytest.raises(ValueError, match="float32 tensor"):
        sample_logits(x[None], u, par)
    for bad in (dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=-0.1),
                dict(min_p=[0.1, 0.2]), dict(min_p=-1e-9)):
        with pytest.raises(ValueError):
            sampling_params(3, device="cpu", **bad)
    lib, p = _lib.load(), ctypes.c_void_p(64)
    bad = _lib.AQ_ERR_VALUE

    def call(rows=1, n=4, ld=0, a=p, b=p, c=p, d=p, e=p, size=1 << 30):
        return lib.aq_sample(a, rows, n, b, c, ld, e, size, d, None, None)
    assert call(rows=-1) == bad and call(n=-1) == bad and call(ld=-1) == bad
    assert call(rows=65536) == bad and call(n=2 ** 31) == bad and call(n=0) == bad
    assert call(ld=3) == bad
    for name in "abcde":
        assert call(**{name: None}) == bad
    size = ctypes.c_size_t()
    assert lib.aq_sample_scratch(3, 5000, ctypes.byref(size)) == _lib.AQ_OK
    assert call(rows=3, n=5000, size=size.value - 1) == bad
    assert call(e=ctypes.c_void_p(68)) == bad
    assert lib.aq_sample_scratch(3, 0, ctypes.byref(size)) == bad
    assert lib.aq_sample_scratch(-1, 5, ctypes.byref(size)) == bad
    assert call(rows=0, a=None, b=None, c=None, d=None) == _lib.AQ_OK


@gpu
def test_refusals_on_the_gpu():
    from alpacca_amd.logits import sample_logits, sampling_params
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    par = sampling_params()
    sample_logits(x, u, par)
    for args in ((x, u.float(), par), (x, u[:1], par), (x, u, par.float()), (x, u, par[:3]),
                 (x, u, par.repeat(3, 1)), (x, u.cpu(), par), (x[:, :0], u, par),
                 (x, u, par.cpu())):
        with pytest.raises(ValueError):
            sample_logits(*args)
    with pytest.raises(ValueError):
        sample_logits(x, u, par, out=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        sample_logits(x, u, par, out=torch.zeros(3, dtype=torch.int64, device="cuda"))
