"""Adjustment of logits (aq_logits_adjust through alpacca_amd.logits): penalties,
biases and masks equal to the definition evaluated in 64 bits and rounded once,
bit for bit; refusals (on the CPU)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from alpacca_amd import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def want64(x, window=None, pen=None, bias=None, allowed=None):
    """The definition, one token after another, in Python floats."""
    rows, n = x.shape
    y = x.astype(np.float64)
    for r in range(rows):
        if window is not None:
            seen = int(window[r, 0])
            toks = window[r, 1:1 + max(0, min(seen, window.shape[1] - 1))]
            rep, pres, freq = (float(p) for p in pen[r])
            for t, c in zip(*np.unique(toks, return_counts=True)):
                if not 0 <= t < n:
                    continue
                v = float(y[r, t])
                with np.errstate(all="ignore"):
                    if rep not in (0.0, 1.0):
                        v = v / rep if v > 0 else v * rep
                    y[r, t] = v - (pres + freq * float(c))
        if bias is not None:
            ids, val, off = bias
            a, b = (0, len(ids)) if off is None else (max(0, int(off[r])),
                                                      min(len(ids), int(off[r + 1])))
            b = max(a, b)  # (a negative end would count from the list's end in Python)
            for t, v in dict(zip(ids[a:b].tolist(), val[a:b].tolist())).items():
                if 0 <= t < n:
                    y[r, t] += v
        if allowed is not None:
            y[r, ~(allowed[r] if allowed.ndim == 2 else allowed)] = -np.inf
    with np.errstate(over="ignore"):
        return y.astype(np.float32)


def dev(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def check(x, window=None, pen=None, bias=None, allowed=None):
    from alpacca_amd.logits import adjust_logits, pack_mask
    mask = None if allowed is None else pack_mask(dev(allowed))
    b = None if bias is None else tuple(dev(t) for t in bias if t is not None)
    want = want64(x, window, pen, bias, allowed)
    xd = dev(x)
    kw = dict(window=dev(window), penalties=dev(pen), bias=b, mask=mask)
    got = adjust_logits(xd, **kw)
    assert np.array_equal(xd.cpu().numpy(), x, equal_nan=True)
    same = adjust_logits(xd, **kw, out=xd)  # in place
    assert same is xd
    for g in (got, same):
        g = g.cpu().numpy()
        assert np.array_equal(g, want, equal_nan=True), np.argwhere(g != want)[:5]


@gpu
@pytest.mark.parametrize("rows,n,last_n", [(1, 1, 1), (1, 31, 3), (3, 1000, 64), (2, 1024, 700),
                                           (5, 1025, 16), (1, 128256, 64), (7, 32003, 3000),
                                           (33, 4099, 40)])
def test_adjust_everything(rows, n, last_n):
    rng = np.random.default_rng(rows + n)
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    window = np.empty((rows, 1 + last_n), np.int64)
    window[:, 0] = rng.integers(0, 2 * last_n + 1, rows)
    window[:, 1:] = (n * rng.random((rows, last_n)) ** 4).astype(np.int64)
    pen = np.stack([rng.uniform(0.8, 1.4, rows), rng.uniform(-1, 1, rows),
                    rng.uniform(-0.5, 0.5, rows)], axis=1)
    sizes = rng.integers(0, 50, rows)
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    ids = rng.integers(0, n, off[-1]).astype(np.int64)
    val = (4 * rng.standard_normal(off[-1])).astype(np.float32)
    allowed = rng.random((rows, n)) < 0.7
    for w in (None, window):
        p = None if w is None else pen
        for b in (None, (ids, val, off)):
            for al in (None, allowed, allowed[0]):
                check(x, w, p, b, al)


@gpu
def test_adjust_edges():
    """Tokens outside the vocabulary, the same token many times in the window
    and twice in the bias list, an empty window, repeat 0 and 1, zero,
    infinite and NaN logits, biases and penalties that are not finite, rows
    whose mask leaves nothing."""
    n, last_n = 70, 9
    x = np.linspace(-5, 5, 6 * n, dtype=np.float32).reshape(6, n)
    x[:, 7] = 0.0
    x[:, 8], x[:, 9], x[:, 10], x[:, 11] = np.inf, -np.inf, np.nan, -0.0
    window = np.zeros((6, 1 + last_n), np.int64)
    window[0] = [20, 3, 3, 3, 3, 3, 7, 8, 9, 10]
    window[1] = [3, -1, n, 2 ** 40, 5, 5, 5, 5, 5, 5]
    window[2] = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9]
    window[3] = [5, 11, 10, 9, 8, 7, 6, 7, 8, 9]
    window[4] = [9, 69, 69, 68, 0, 0, 0, 33, 32, 31]
    window[5] = [-4, 1, 2, 3, 4, 5, 6, 7, 8, 9]
    pen = np.array([[1.1, 0.5, 0.25], [0.0, 1.0, 0.0], [1.3, 1, 1], [1.0, 0.0, 0.5],
                    [2.0, np.inf, 0.0], [1.5, 1, 1]])
    ids = np.array([3, 3, 70, -1, 8, 9, 2, 3, 12, 2 ** 33], np.int64)
    val = np.array([1, 2, 9, 9, -np.inf, 3, np.nan, 0.5, 3e38, 1], np.float32)
    off = np.array([0, 4, 4, 8, 9, 99, 10], np.int64)
    off[3] = -5  # clipped to the list
    allowed = np.ones((6, n), bool)
    allowed[1] = False
    allowed[4, 1:] = False
    for b in (None, (ids, val, None), (ids, val, off)):
        for al in (None, allowed, np.zeros(n, bool)):
            check(x, window, pen, b, al)
    check(x, None, None, (ids[:0], val[:0], None), None)


@gpu
def test_one_dimension_streams_and_capture():
    from alpacca_amd.logits import adjust_logits, pack_mask
    rng = np.random.default_rng(1)
    n = 5000
    x = rng.standard_normal((1, n)).astype(np.float32)
    window = np.array([[4, 5, 6, 6, 7]], np.int64)
    pen = np.array([[1.2, 0.1, 0.2]])
    allowed = rng.random(n) < 0.5
    want = want64(x, window, pen, None, allowed)[0]
    kw = dict(window=dev(window[0]), penalties=dev(pen[0]), mask=pack_mask(dev(allowed)))
    xd, out = dev(x[0]), torch.empty(n, device="cuda")
    assert np.array_equal(adjust_logits(xd, **kw).cpu().numpy(), want)
    assert np.array_equal(adjust_logits(dev(np.repeat(x[0], 2))[::2], **kw).cpu().numpy(), want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        adjust_logits(xd, **kw, out=out)
    for i in range(3):
        with torch.cuda.stream(s):
            out.zero_()
            xd.copy_(dev(x[0]) + i)
            g.replay()
        s.synchronize()
        assert np.array_equal(out.cpu().numpy(),
                              want64((x + np.float32(i)), window, pen, None, allowed)[0])


def test_pack_mask():
    from alpacca_amd.logits import pack_mask
    rng = np.random.default_rng(0)
    for shape in ((1,), (31,), (32,), (33,), (3, 70)):
        a = torch.from_numpy(rng.random(shape) < 0.5)
        w = pack_mask(a).numpy().view(np.uint32)
        back = (w[..., :, None] >> np.arange(32, dtype=np.uint32)) & 1
        back = back.reshape(*w.shape[:-1], -1)
        assert np.array_equal(back[..., :shape[-1]].astype(bool), a.numpy())
        assert not back[..., shape[-1]:].any()
    with pytest.raises(ValueError):
        pack_mask(torch.zeros(3))


def test_c_refusals():
    lib = _lib.load()

    def adjust(x=4096, rows=2, n=100, window=None, last_n=0, pen=None, ids=None, bias=None,
               off=None, n_bias=0, mask=None, ld=0, out=4096):
        return lib.aq_logits_adjust(x, rows, n, window, last_n, pen, ids, bias, off, n_bias, mask,
                                    ld, out, None)
    bad = [adjust(rows=-1), adjust(n=-1), adjust(rows=65536), adjust(window=8, last_n=4),
           adjust(pen=8), adjust(window=8, pen=8, last_n=0), adjust(n_bias=1, ids=8),
           adjust(n_bias=1, bias=8), adjust(n_bias=-1), adjust(mask=8, ld=3), adjust(x=None),
           adjust(out=None), adjust(out=4100), adjust(out=4096 - 4), adjust(n=2 ** 33)]
    assert all(rc == _lib.AQ_ERR_VALUE for rc in bad), bad
    assert adjust(rows=0, x=None, out=None) == adjust(n=0) == _lib.AQ_OK


@gpu
def test_python_refusals():
    from alpacca_amd.logits import adjust_logits
    x = torch.zeros(2, 40, device="cuda")
    w = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    p = torch.zeros(2, 3, dtype=torch.float64, device="cuda")
    m = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    i, v = w[0], x[0, :5]
    for bad in (lambda: adjust_logits(x.cpu()), lambda: adjust_logits(x.half()),
                lambda: adjust_logits(x, window=w), lambda: adjust_logits(x, penalties=p),
                lambda: adjust_logits(x, window=w[:1], penalties=p),
                lambda: adjust_logits(x, window=w.int(), penalties=p),
                lambda: adjust_logits(x, window=w, penalties=p.float()),
                lambda: adjust_logits(x, window=w[:, :1], penalties=p),
                lambda: adjust_logits(x, mask=m[:, :1]), lambda: adjust_logits(x, mask=m[:1]),
                lambda: adjust_logits(x, mask=m.long()), lambda: adjust_logits(x, mask=m.cpu()),
                lambda: adjust_logits(x, bias=(i, v[:4])), lambda: adjust_logits(x, bias=i),
                lambda: adjust_logits(x, bias=(i, v, i[:2])), lambda: adjust_logits(x, out=x[:1]),
                lambda: adjust_logits(x, out=x.t())):
        with pytest.raises(ValueError):
            bad()
    assert adjust_logits(x[:0]).shape == (0, 40)


@gpu
def test_bias_offsets_past_the_list():
    """Offsets are clipped to the list, the largest 64-bit ones too: such a row
    owns no entry, or all from its start on."""
    big = 2 ** 63 - 1
    rows, n = 5, 1500
    x = np.linspace(-2, 2, rows * n, dtype=np.float32).reshape(rows, n)
    ids = np.arange(0, 1200, 2, dtype=np.int64)
    val = np.linspace(-1, 1, 600, dtype=np.float32)
    for off in ([big, big, big - 300, 590, big, big], [-big - 1, big, 0, 3, big, -big - 1],
                [590, big, 599, big - 1200, 600, 601]):
        check(x, None, None, (ids, val, np.array(off, np.int64)), None)


def batch_inputs(rng, rows, n, last_n):
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    window = np.empty((rows, 1 + last_n), np.int64)
    window[:, 0] = rng.integers(0, 2 * last_n + 1, rows)
    window[:, 1:] = (n * rng.random((rows, last_n)) ** 3).astype(np.int64)
    pen = np.stack([rng.uniform(0.8, 1.4, rows), rng.uniform(-1, 1, rows),
                    rng.uniform(-0.5, 0.5, rows)], axis=1)
    off = np.concatenate([[0], np.cumsum(rng.integers(0, 1500, rows))]).astype(np.int64)
    ids = rng.integers(0, n, off[-1]).astype(np.int64)
    val = (4 * rng.standard_normal(off[-1])).astype(np.float32)
    allowed = rng.random((rows, n)) < 0.6
    allowed[rows // 2] = False
    return x, window, pen, (ids, val, off), allowed


@gpu
@pytest.mark.parametrize("rows,n,last_n", [(64, 32771, 700), (33, 65537, 1500), (1025, 1999, 40),
                                           (1024, 2048, 70), (512, 2049, 70), (16, 131073, 64)])
def test_adjust_large_batches(rows, n, last_n):
    """From 1024 slices of 2048 logits on (rows x n): windows, ragged biases of
    more entries than a workgroup has threads, a mask per row that leaves one
    with nothing."""
    rng = np.random.default_rng(rows + n)
    assert rows * -(-n // 2048) >= 1024
    x, window, pen, bias, allowed = batch_inputs(rng, rows, n, last_n)
    x[:, ::97] = np.inf
    x[:, 5::89] = np.nan
    check(x, window, pen, bias, allowed)
    check(x, None, None, bias, allowed[0])
    check(x, window, pen, None, None)


@gpu
@pytest.mark.parametrize("n", [32771, 4099])
def test_adjust_rows_alone_and_in_batches(n):
    """A row's logits are the same bits in a batch on either side of the border
    between the slices' sizes, and alone."""
    from alpacca_amd.logits import adjust_logits, pack_mask
    words = -(-n // 2048)
    above = -(-1024 // words)
    rng = np.random.default_rng(n)
    x, window, pen, (ids, val, off), allowed = batch_inputs(rng, above, n, 200)

    def run(rows, out_of_place):
        xd = dev(x[:rows])
        return adjust_logits(xd, window=dev(window[:rows]), penalties=dev(pen[:rows]),
                             bias=(dev(ids), dev(val), dev(off[:rows + 1])),
                             mask=pack_mask(dev(allowed[:rows])),
                             out=None if out_of_place else xd).view(torch.int32)
    assert above * words >= 1024 > (above - 1) * words
    for fresh in (True, False):
        many, fewer, one = (run(rows, fresh) for rows in (above, above - 1, 1))
        assert torch.equal(many[:-1], fewer) and torch.equal(many[:1], one)
