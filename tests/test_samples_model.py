"""Model.generate_samples: every drawn token against the float32 oracle whose decode
attention reads keys and values rounded as the pages hold them, the same tokens
whatever runs beside a sequence or how the step is run, refusals.

Tolerance.  Quantized against float32 models agree to 1e-2 of the largest logit
(the bar of the other model tests); the pages' rounding, 2^-11 (fp16) or 2^-8
(bf16) of each value, is in the oracle too, so what is left of it are values next to
a half step.  Logits off by e move every weight's share by the factor e^(2 e / T) at
most, and with it the place of a border between two tokens in [0, 1]."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest

from oracle import model_ref as MR
from tests.test_kv8 import coded, values64
from tests.test_sample import kept_of

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def tiny(**kw):
    from alpacca_amd.model import synthetic_llama_1b
    args = dict(seed=10, n_layer=2, n_embd=256, n_head=4, n_kv=2, n_ff=512, n_vocab=500,
                n_ctx_train=256, std=0.05)
    args.update(kw)
    return synthetic_llama_1b(**args)


def rounded(x, kind):
    x = torch.from_numpy(np.ascontiguousarray(x, np.float32))
    return x.to(torch.float16 if kind == "f16" else torch.bfloat16).float().numpy()


def oracle(hp, tensors, kind, monkeypatch, kv_dtype="f32"):
    """RefModel whose single-token attention reads rounded keys and values (and
    the prompt's, over an 8-bit cache, coded ones)."""
    one, batch = MR.attention_np, MR.attention_batch_np
    monkeypatch.setattr(MR, "attention_np",
                        lambda q, K, V, *a: one(q, rounded(K, kind), rounded(V, kind), *a))
    if kv_dtype == "q8":
        def c(x):
            return values64(*coded(x)).astype(np.float32)
        monkeypatch.setattr(MR, "attention_batch_np",
                            lambda q, K, V, *a: batch(q, c(K), c(V), *a))
    return MR.RefModel(hp, tensors)


def check_tokens(ref, prompt, out, U, par, edit=lambda x: x):
    for r, toks in enumerate(out):
        ref.reset()
        logits = ref.prefill(prompt)
        for i, t in enumerate(toks):
            x = edit(np.asarray(logits, np.float32))
            temp, k, p, min_p = (float(v[r]) if np.ndim(v) else float(v) for v in par)
            err = 1e-2 * np.abs(logits).max()
            if not temp > 0:
                assert x[t] >= x.max() - 2 * err, (r, i)
            else:
                # what k, p and min-p keep moves with the logits as well: the token's
                # place among all that could be kept, and among the least
                slack = np.expm1(2 * err / temp)
                o, w = kept_of(x, temp, k, p, min_p)
                run = np.concatenate([[0], np.cumsum(w)]) / w.sum()
                near = np.flatnonzero(np.abs(x[o] - x[t]) <= 2 * err)
                if near.size == 0:  # at the kept set's end
                    assert x[t] >= x[o[-1]] - 2 * err, (r, i)
                    near = np.array([len(o) - 1])
                u = float(U[i, r])
                assert run[near[0]] - slack <= u <= run[near[-1] + 1] + slack, (r, i, u)
            if i + 1 < len(toks):
                logits = ref.forward(t)


SETTINGS = dict(temperature=[0.8, 1.0, 0.0, 0.6, 1.2], top_k=[40, 0, 0, 5, 0],
                top_p=[0.9, 1.0, 1.0, 1.0, 0.7], min_p=[0.0, 0.02, 0.0, 0.0, 0.0])


@gpu
@pytest.mark.parametrize("shape,style,n_rot,kind,n_p,graph,kv_dtype", [
    (dict(), "norm", None, "f16", 50, True, "f32"),
    (dict(n_embd=512, n_head=4, n_kv=1), "neox", None, "bf16", 64, True, "f32"),
    (dict(n_embd=768, n_head=12, n_kv=4), "neox", 20, "f16", 33, True, "q8"),
    (dict(n_embd=512, n_head=2, n_kv=1), "norm", 20, "f16", 1, False, "q8")])
def test_tokens(monkeypatch, shape, style, n_rot, kind, n_p, graph, kv_dtype):
    """(Groups of 3 and heads of 256 are what the 8-bit cache takes the prompt of.)"""
    from alpacca_amd.model import Model
    hp, tensors = tiny(**shape)
    hp = dataclasses.replace(hp, rope_style=style, n_rot=n_rot or hp.head_dim)
    prompt = [int(t) for t in np.random.default_rng(5).integers(0, hp.n_vocab, n_p)]
    m = Model(hp, tensors, kv_dtype=kv_dtype)
    n_seq, n_gen = 5, 40
    timing = {}
    out = m.generate_samples(prompt, n_gen, n_seq, seed=3, kv_dtype=kind, page_size=32, graph=graph,
                             timing=timing, **SETTINGS)
    assert len(out) == n_seq and all(len(o) == n_gen for o in out)
    assert timing["steps"] == n_gen - 1 and timing["gen_ms"] > 0
    assert m.cached_ids == prompt and m.n_past == n_p
    U = torch.rand(n_gen, n_seq, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    check_tokens(oracle(hp, tensors, kind, monkeypatch, kv_dtype), prompt, out, U,
                 [SETTINGS[k] for k in ("temperature", "top_k", "top_p", "min_p")])
    assert len({tuple(o) for o in out}) == n_seq


@gpu
def test_same_tokens_with_and_without_graph_and_after_other_calls():
    from alpacca_amd.model import Model
    hp, tensors = tiny()
    prompt = [int(t) for t in np.random.default_rng(6).integers(0, hp.n_vocab, 70)]
    m = Model(hp, tensors)
    greedy = m.generate_greedy(prompt, 30)
    a = m.generate_samples(prompt, 60, 7, seed=1, **{k: v + v[:2] for k, v in SETTINGS.items()})
    b = m.generate_samples(prompt, 60, 7, seed=1, graph=False,
                           **{k: v + v[:2] for k, v in SETTINGS.items()})
    assert a == b
    # the model's cache holds the prompt, as after prefill: what repeats it goes on there
    ref = Model(hp, tensors)
    ref.prefill(prompt)
    assert np.array_equal(m.prefill(prompt + [5]), ref.prefill(prompt + [5]))
    assert m.generate_greedy(prompt, 30) == greedy
    # in chunks, from the 8-bit cache, one token, one sequence
    m.prefill_chunk = 16
    assert m.generate_samples(prompt, 60, 7, seed=1,
                              **{k: v + v[:2] for k, v in SETTINGS.items()}) == a
    q8 = Model(hp, tensors, kv_dtype="q8")
    assert len(q8.generate_samples(prompt, 9, 3)) == 3
    assert [len(o) for o in m.generate_samples(prompt, 1, 4)] == [1] * 4
    one = m.generate_samples(prompt, 12, 1, temperature=0.0)[0]
    assert len(one) == 12 and one[0] == greedy[0]
    assert m.generate_samples(prompt, 20, 2, seed=1) != m.generate_samples(prompt, 20, 2, seed=2)


@gpu
def test_bias_and_allowed(monkeypatch):
    from alpacca_amd.model import Model
    hp, tensors = tiny()
    rng = np.random.default_rng(9)
    prompt = [int(t) for t in rng.integers(0, hp.n_vocab, 20)]
    allowed = rng.random(hp.n_vocab) < 0.2
    bias = {int(t): float(v) for t, v in zip(rng.permutation(hp.n_vocab)[:30],
                                             2 * rng.standard_normal(30))}
    out = Model(hp, tensors).generate_samples(prompt, 25, 4, seed=2, logit_bias=bias,
                                              allowed=allowed)
    assert allowed[np.array(out)].all()

    def edit(x):
        x = x.copy()
        for t, v in bias.items():
            x[t] += np.float32(v)
        x[~allowed] = -np.inf
        return x
    U = torch.rand(25, 4, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    check_tokens(oracle(hp, tensors, "f16", monkeypatch), prompt, out, U, (1.0, 0, 1.0, 0.0), edit)


@gpu
def test_refusals():
    from alpacca_amd.model import Model
    hp, tensors = tiny()
    m = Model(hp, tensors)
    for kw in (dict(prompt=[]), dict(n_gen=0), dict(n_seq=0), dict(kv_dtype="f32"),
               dict(page_size=20), dict(temperature=float("nan")), dict(top_k=-1),
               dict(top_p=[0.5, 0.5, 0.5]), dict(min_p=-0.5), dict(allowed=np.zeros(500, bool))):
        with pytest.raises(ValueError):
            m.generate_samples(**{**dict(prompt=[1, 2], n_gen=3, n_seq=2), **kw})
    for tok in (-1, 500):
        with pytest.raises(IndexError):
            m.generate_samples([1, tok], 3)
    with pytest.raises(RuntimeError, match="context window full"):
        m.generate_samples([1] * 250, 8)
    assert len(m.generate_samples([1] * 250, 7)[0]) == 7
    small = tiny(n_embd=256, n_head=8)  # heads of 32
    from alpacca_amd.kvcache import check_paged_heads
    with pytest.raises(ValueError, match="paged KV cache takes"):
        check_paged_heads(8, 2, 32)
    with pytest.raises((ValueError, RuntimeError)):
        Model(*small).generate_samples([1, 2], 3)


def test_heads():
    from alpacca_amd.kvcache import HEAD_DIMS, MAX_GROUP, check_paged_heads
    for hd in HEAD_DIMS:
        check_paged_heads(MAX_GROUP * 3, 3, hd)
        for n_head, n_kv in ((MAX_GROUP * 3 + 3, 3), (7, 2), (2, 4), (0, 1)):
            with pytest.raises(ValueError):
                check_paged_heads(n_head, n_kv, hd)


def test_page_sizes():
    from alpacca_amd.kvcache import check_page_size
    for size in (32, 64, 96, 65536):
        check_page_size(size)
    for size in (0, -64, 20, 31, 33, 65568, 1 << 40):
        with pytest.raises(ValueError, match="multiple of 32"):
            check_page_size(size)


@gpu
@pytest.mark.parametrize("size", [0, -64, 33, 1 << 20])
def test_bad_page_size_leaves_the_cache(size):
    """Refused before the model's own cache is emptied."""
    from alpacca_amd.model import Model
    m = Model(*tiny())
    m.generate_greedy([1, 2, 3], 2)
    n_past = m.n_past
    with pytest.raises(ValueError, match="multiple of 32"):
        m.generate_samples([1, 2], 3, page_size=size)
    assert m.n_past == n_past > 0
