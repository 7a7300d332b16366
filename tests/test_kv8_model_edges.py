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


def test_allowed_tokens_that_are_banned():
    """A token outside the mask is never returned: refused before the first
    step where every allowed token's bias is -inf, and a RuntimeError where
    the penalties leave no allowed logit above -inf."""
    hp, tensors = tiny()
    m = model(hp, tensors)
    ban = float("-inf")

    def only(*ids):
        a = np.zeros(hp.n_vocab, bool)
        a[list(ids)] = True
        return a
    for graph in (True, False):
        with pytest.raises(ValueError, match="allowed"):
            m.generate_greedy([1, 2], 4, graph=graph, allowed=only(5), logit_bias={5: ban})
        with pytest.raises(ValueError, match="allowed"):
            m.generate_greedy([1, 2], 4, graph=graph, allowed=only(5, 9),
                              logit_bias={9: ban, 5: ban, 3: 1.0})
        assert m.generate_greedy([1, 2], 4, graph=graph, allowed=only(5, 9),
                                 logit_bias={9: ban}) == [5] * 4
        # each said token falls to -inf: two steps leave nothing, one token more fails
        kw = dict(graph=graph, allowed=only(5, 9), presence_penalty=1e39)
        assert sorted(m.generate_greedy([1, 2], 2, **kw)) == [5, 9]
        with pytest.raises(RuntimeError, match="allowed"):
            m.generate_greedy([1, 2], 3, **kw)
        assert m.n_past == 0 and m.cached_ids == []
    # the model is as it was
    want = model(hp, tensors).generate_greedy([1, 2], 6)
    assert m.generate_greedy([1, 2], 6) == want


def test_biases_past_float32():
    hp, tensors = tiny()
    m = model(hp, tensors)
    for v in (1e39, -1e39):
        with pytest.raises(ValueError, match="float32"):
            m.generate_greedy([1, 2], 2, logit_bias={3: v})
    assert m.generate_greedy([1, 2], 2, logit_bias={3: float("inf")}) == [3, 3]


def test_scratch_is_shared_and_counted():
    """A model's layers share one scratch; a cache of its own has another."""
    from alpacca_amd.kvcache import QuantKVCache
    hp, tensors = tiny(n_layer=3)
    kv8 = model(hp, tensors, kv_dtype="q8").kv8
    assert len({c._scratch.data_ptr() for c in kv8}) == 1
    for hd, mb in ((64, 18), (128, 35), (256, 68)):
        a = QuantKVCache(2, 40, hd)
        b = QuantKVCache(1, 70, hd, scratch=a)
        assert a.scratch_nbytes() == b.scratch_nbytes() == 65536 * (hd + 4) * 4
        assert round(a.scratch_nbytes() / 1e6) == mb
        assert a.storage_nbytes() == 2 * (2 * 2 * 32 * hd + 2 * 2 * 4 + 2 * 32 * hd * 4 + 16)
        assert a._scratch.data_ptr() == b._scratch.data_ptr() != QuantKVCache(
            2, 40, hd)._scratch.data_ptr()
