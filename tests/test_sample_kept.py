"""Sampling: what top-p keeps of a top-k where few blocks of 64 tokens hold anything,
and min-p ends before the k-th token (the kernel's list of a row goes by its blocks'
largest logits, of which there may be fewer than k).  Tolerances: those of
tests/test_sample.py, whose check() this uses."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_sample import check, dev, kept_of

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def sixteen_blocks():
    """1000 logits: the blocks' largest from 2 to 3, 32 tokens just below these."""
    x = np.full(1000, -9.0, np.float32)
    x[::64] = np.linspace(2, 3, 16)
    x[1::64] = 1.9
    x[2::64] = 1.8
    return x


def test_sixteen_blocks_by_hand():
    """The 40 largest sum to 17.9, of which 0.6 is more than the 14 tokens above 0.4
    sum to: min-p's end counts."""
    x = sixteen_blocks()
    o, w = kept_of(x, 1.0, 40, 1.0, 0.0)
    assert len(o) == 40 and abs(w.sum() - 17.9) < 0.01
    kept, w = kept_of(x, 1.0, 40, 0.6, 0.4)
    assert len(kept) == 14 and abs(w.sum() - 9.41) < 0.01
    assert np.searchsorted(np.cumsum(w), 0.5 * w.sum(), side="right") == 5  # the order's 6th


@gpu
def test_sixteen_blocks():
    rows = 97
    x = np.tile(sixteen_blocks(), (rows, 1))
    u = (np.arange(rows) + 0.5) / rows
    for p in (0.3, 0.5, 0.6, 0.9):
        check(x, u, (1.0, 40, p, 0.4))
    from alpacca_amd.logits import sample_logits
    tok = sample_logits(dev(x), dev(u), dev(np.array([1.0, 40, 0.6, 0.4]))).cpu().numpy()
    assert len(set(tok.tolist())) == 14


@gpu
@pytest.mark.parametrize("temp", [1.0, 1.3])
@pytest.mark.parametrize("k", [100, 300, 500])
@pytest.mark.parametrize("n", [1000, 2000, 4000, 4097, 9600])
def test_more_than_the_blocks(n, k, temp):
    """Near-flat rows, top-k above the number of blocks or near it."""
    rng = np.random.default_rng(n + k)
    rows = 12
    for p in (0.5, 0.6, 0.9, 0.999):
        for min_p in (0.05, 0.1, 0.2):
            check(rng.standard_normal((rows, n)).astype(np.float32), rng.random(rows),
                  (temp, k, p, min_p))


@gpu
@pytest.mark.parametrize("n", [3001, 32003, 128256])
@pytest.mark.parametrize("m", [1, 30, 45, 200, 700, 2000, 3000])
def test_few_tokens_left(n, m):
    """Rows of which a mask leaves m tokens, side by side or scattered."""
    rng = np.random.default_rng(n + m)
    rows = 6
    x = np.full((rows, n), -np.inf, np.float32)
    for r in range(rows):
        first = int(rng.integers(0, n - m + 1))
        at = np.arange(first, first + m) if r % 2 else rng.choice(n, m, replace=False)
        x[r, at] = rng.standard_normal(m) * (0.5 if r < 4 else 2.0)
    for par in ((0.8, 40, 0.95, 0.05), (1.0, 40, 0.6, 0.4), (1.0, m, 0.6, 0.2),
                (1.3, m + 1, 0.5, 0.1), (1.0, max(m // 2, 1), 0.9, 0.1), (2.0, 1000, 0.7, 0.3),
                (30.0, 2 * m, 0.99, 0.5), (1.0, 40, 1.0, 0.4)):
        check(x, rng.random(rows), par)


@gpu
def test_lowest_floats_among_few():
    """Masked by the type's lowest value: tokens of the order, of no weight."""
    rng = np.random.default_rng(2)
    for n in (900, 4096, 9600):
        x = np.full((8, n), np.finfo(np.float32).min, np.float32)
        for r in range(8):
            x[r, 100:100 + 60 * (r + 1)] = rng.standard_normal(60 * (r + 1))
        for par in ((1.0, 300, 0.6, 0.2), (1.3, 700, 0.5, 0.1), (0.7, 899, 0.9, 0.3)):
            check(x, rng.random(8), par)


@gpu
def test_generated_with_all_settings_and_allowed(monkeypatch):
    """The settings together in generation, where `allowed` leaves tokens of eight
    blocks and top-k asks for more."""
    from alpacca_amd.model import Model
    from tests.test_samples_model import check_tokens, oracle, tiny
    hp, tensors = tiny()
    rng = np.random.default_rng(12)
    prompt = [int(t) for t in rng.integers(0, hp.n_vocab, 20)]
    allowed = rng.random(hp.n_vocab) < 0.3
    par = dict(temperature=[1.0, 1.5, 0.8, 1.2], top_k=[60, 100, 40, 30],
               top_p=[0.6, 0.5, 0.95, 0.8], min_p=[0.1, 0.2, 0.05, 0.15])
    m = Model(hp, tensors)
    out = m.generate_samples(prompt, 25, 4, seed=4, allowed=allowed, **par)
    assert allowed[np.array(out)].all()
    assert m.generate_samples(prompt, 25, 4, seed=4, allowed=allowed, graph=False, **par) == out

    def edit(x):
        return np.where(allowed, x, np.float32(-np.inf))
    U = torch.rand(25, 4, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    check_tokens(oracle(hp, tensors, "f16", monkeypatch), prompt, out, U,
                 [par[k] for k in ("temperature", "top_k", "top_p", "min_p")], edit)
