"""The decode and prefill steps of Model over the 8-bit KV cache, and greedy
generation with adjusted logits: against the float32 oracle whose attention
reads keys and values coded as the cache codes them, against the same steps
taken one by one, and against the adjustment evaluated in 64 bits."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest

from oracle import model_ref as MR
from tests.test_kv8 import coded, values64
from tests.test_logits import want64

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def model(hp, tensors, **kw):
    from alpacca_amd.model import Model
    return Model(hp, tensors, **kw)


def tiny(**kw):
    from alpacca_amd.model import synthetic_llama_1b
    args = dict(seed=10, n_layer=2, n_embd=256, n_head=4, n_kv=2, n_ff=512, n_vocab=500,
                n_ctx_train=256, std=0.05)
    args.update(kw)
    return synthetic_llama_1b(**args)


@pytest.fixture()
def coded_oracle(monkeypatch):
    """RefModel with its attention over coded keys and values."""
    one, batch = MR.attention_np, MR.attention_batch_np

    def c(x):
        return values64(*coded(x)).astype(np.float32)
    monkeypatch.setattr(MR, "attention_np", lambda q, K, V, *a: one(q, c(K), c(V), *a))
    monkeypatch.setattr(MR, "attention_batch_np",
                        lambda q, K, V, *a: batch(q, c(K), c(V), *a))
    return MR.RefModel


SHAPES = [dict(), dict(n_embd=512, n_head=4, n_kv=1), dict(n_embd=768, n_head=12, n_kv=4),
          dict(n_embd=512, n_head=2, n_kv=1)]  # groups of 2, 4 and 3; heads of 64, 128, 64, 256


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("style,n_rot,fused", [("norm", None, True), ("neox", None, True),
                                               ("neox", 20, True), ("norm", 20, False)])
def test_logits(coded_oracle, shape, style, n_rot, fused):
    """Prompt in one chunk, then single tokens through a block's border: the
    logits within 1e-2 of their largest (the bar of quantized against float32
    models; a key or value next to a half step may be coded a step apart,
    1/127 of its block's largest)."""
    hp, tensors = tiny(**shape)
    hp = dataclasses.replace(hp, rope_style=style, n_rot=n_rot or hp.head_dim)
    toks = [int(t) for t in np.random.default_rng(5).integers(0, hp.n_vocab, 70)]
    m, ref = model(hp, tensors, kv_dtype="q8", fused=fused), coded_oracle(hp, tensors)
    a, b = m.prefill(toks[:60]), ref.prefill(toks[:60])
    assert np.abs(a - b).max() < 1e-2 * np.abs(b).max()
    for t in toks[60:]:
        a, b = m.forward(t), ref.forward(t)
        assert np.abs(a - b).max() < 1e-2 * np.abs(b).max()


@pytest.mark.parametrize("graph,batch_prefill", [(True, True), (True, False), (False, True)])
def test_greedy_tokens(coded_oracle, graph, batch_prefill):
    """Greedy tokens equal the oracle's up to a step whose two largest logits
    are within 2 % of the largest."""
    hp, tensors = tiny()
    prompt = [int(t) for t in np.random.default_rng(5).integers(0, hp.n_vocab, 50)]
    m, ref = model(hp, tensors, kv_dtype="q8"), coded_oracle(hp, tensors)
    got = m.generate_greedy(prompt, 90, graph=graph, batch_prefill=batch_prefill)
    assert m.n_past == 139 and len(got) == 90
    if batch_prefill:
        logits = ref.prefill(prompt)
    else:
        for t in prompt:
            logits = ref.forward(t)
    sure = 0
    for t in got:
        top = np.sort(logits)[-2:]
        if top[1] - top[0] < 0.02 * np.abs(logits).max():
            break
        assert int(np.argmax(logits)) == t, sure
        sure += 1
        logits = ref.forward(t)
    print(f"{sure} tokens compared", flush=True)
    assert sure >= 3


def test_going_back_is_as_if_never():
    """A prompt that repeats part of the cached one: inside the last block and
    from an earlier one (which starts at its first position), the same bits
    as without what was dropped."""
    hp, tensors = tiny()
    toks = [int(t) for t in np.random.default_rng(6).integers(0, hp.n_vocab, 70)]
    m = model(hp, tensors, kv_dtype="q8")
    m.prefill(toks, batch=False)
    for keep in (66, 40, 33, 32, 1):
        new = toks[:keep] + [7, 8, (toks[min(keep, 69)] + 1) % hp.n_vocab]
        got = m.prefill(new, batch=False)
        assert m.n_past == len(new) and m.cached_ids == new
        fresh = model(hp, tensors, kv_dtype="q8")
        assert np.array_equal(got, fresh.prefill(new, batch=False)), keep
        for a, b in zip(m.kv8, fresh.kv8):
            a.length = b.length = len(new)
            for x, y in zip(a.read(), b.read()):
                assert torch.equal(x, y), keep
        m.prefill(toks, batch=False)


def test_batched_prompt_in_chunks():
    """A prompt in ragged chunks equals it whole within the coding's error
    (a query of a longer chunk sees its own block coded with more tokens)."""
    hp, tensors = tiny()
    toks = [int(t) for t in np.random.default_rng(8).integers(0, hp.n_vocab, 150)]
    whole = model(hp, tensors, kv_dtype="q8").prefill(toks)
    for chunk in (1, 7, 64):
        m = model(hp, tensors, kv_dtype="q8")
        m.prefill_chunk = chunk
        got = m.prefill(toks)
        assert np.abs(got - whole).max() < 3e-2 * np.abs(whole).max()


@pytest.mark.parametrize("kv_dtype", ["f32", "q8"])
@pytest.mark.parametrize("kind", ["all", "bias", "mask", "window"])
def test_generate_with_adjusted_logits(kv_dtype, kind):
    """Captured generation (single and several steps per graph) equals single
    forward steps whose logits are adjusted on the host in 64 bits."""
    hp, tensors = tiny()
    rng = np.random.default_rng(9)
    prompt = [int(t) for t in rng.integers(0, hp.n_vocab, 20)]
    pres, freq, rep, last_n = 0.7, 0.3, 1.2, 24
    bias = {int(t): float(v) for t, v in zip(rng.permutation(hp.n_vocab)[:30],
                                             rng.standard_normal(30))}
    allowed = rng.random(hp.n_vocab) < 0.3
    if kind in ("bias", "mask"):
        pres = freq = 0.0
        rep = 1.0
    if kind in ("mask", "window"):
        bias = None
    if kind in ("bias", "window"):
        allowed = None
    a = model(hp, tensors, kv_dtype=kv_dtype)
    got = a.generate_greedy(prompt, 80, batch_prefill=False, repeat_penalty=rep,
                            repeat_last_n=last_n, presence_penalty=pres, frequency_penalty=freq,
                            logit_bias=bias, allowed=allowed)
    b = model(hp, tensors, kv_dtype=kv_dtype)
    logits = b.prefill(prompt, batch=False)
    said, want = list(prompt), []
    for i in range(80):
        window = np.array([[min(len(said), last_n)] + (said[-last_n:] + [0] * last_n)[:last_n]])
        listed = None
        if bias:
            listed = (np.array(list(bias)), np.array(list(bias.values()), np.float32), None)
        use = kind in ("all", "window")
        y = want64(logits[None], window if use else None, np.array([[rep, pres, freq]]), listed,
                   allowed)
        want.append(int(np.argmax(y[0])))
        said.append(want[-1])
        if i < 79:
            logits = b.forward(want[-1])
    assert got == want
    if allowed is not None:
        assert allowed[got].all()
    # a second call without any of it is not touched by the first
    assert a.generate_greedy(prompt, 10) == model(hp, tensors, kv_dtype=kv_dtype).generate_greedy(
        prompt, 10)


def test_refusals():
    hp, tensors = tiny()
    with pytest.raises(ValueError, match="kv_dtype"):
        model(hp, tensors, kv_dtype="q4")
    m = model(hp, tensors, kv_dtype="q8")
    for kw in (dict(allowed=np.zeros(500, bool)), dict(allowed=np.ones(499, bool)),
               dict(allowed=np.ones(500)), dict(presence_penalty=float("nan")),
               dict(frequency_penalty=float("inf")), dict(logit_bias={3: float("nan")})):
        with pytest.raises(ValueError):
            m.generate_greedy([1, 2], 3, **kw)
    with pytest.raises(IndexError):
        m.generate_greedy([1, 2], 3, logit_bias={500: 1.0})
    small = tiny(n_embd=256, n_head=8)  # heads of 32
    with pytest.raises(ValueError):
        model(*small, kv_dtype="q8")
