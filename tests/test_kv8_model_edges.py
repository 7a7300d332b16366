"""Model on the 8-bit KV cache and greedy generation with adjusted logits at
their edges: a prompt that goes back after one that failed, shapes that the
cache does not take, masks whose tokens are all banned."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest

from tests.test_kv8_model import model, tiny

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("batch", [True, False])
@pytest.mark.parametrize("cut", [64, 65])
def test_going_back_after_a_refused_prompt(batch, cut):
    """A prompt with a token out of range is refused after its common part has
    shortened the cached one; what follows is as if it had never been."""
    hp, tensors = tiny()
    toks = [int(t) for t in np.random.default_rng(6).integers(0, hp.n_vocab, 70)]
    for keep in (cut, 60, 33, 20):
        m = model(hp, tensors, kv_dtype="q8")
        m.prefill(toks, batch=False)
        with pytest.raises(IndexError):
            m.prefill(toks[:cut] + [hp.n_vocab], batch=batch)
        assert m.n_past == len(m.cached_ids) <= cut
        new = toks[:keep] + [7, 8, (toks[keep] + 1) % hp.n_vocab]
        got = m.prefill(new, batch=False)
        fresh = model(hp, tensors, kv_dtype="q8")
        assert np.array_equal(got, fresh.prefill(new, batch=False)), keep
        for a, b in zip(m.kv8, fresh.kv8):
            a.length = b.length = len(new)
            for x, y in zip(a.read(), b.read()):
                assert torch.equal(x, y), keep
