"""Measured cases of the 8-bit KV cache and of the adjustment of logits.

The operators are steps of one generated token (or prompt) of a served model:

* ``store``: rotate the queries and keys of t tokens, code keys and values to
  int8 and put them into the cache, and read back the blocks that changed;
* ``attend``: grouped-query causal attention of t tokens over the cache;
* ``step``: one token's rotation, store and attention in one call, as a
  decode step makes it for each layer;
* ``logits``: penalties for tokens already said, per-token biases and a
  grammar's mask on the logits of each row.

The cache codes blocks of 32 positions of one kv head (K and V apart): with
amax the largest magnitude among the tokens the block holds so far, the scale
is s = fl32(amax / 127) and each value x is held as the whole number nearest to
x / s (ties to even), standing for s times that.  Keys are coded after their
rotation, which rounds each product and each difference to fp32.

With ``own`` false, ``run`` computes the operators with elementary torch
operations; with ``own`` true through alpacca_amd.kvcache and
alpacca_amd.logits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
ROPE_BASE = 500000.0


# ---- the cases ---------------------------------------------------------------

def listed():
    heads_1b = dict(n_head=32, n_kv=8, head_dim=64, neox=False)
    heads_8b = dict(n_head=32, n_kv=8, head_dim=128, neox=False)
    return [
        # one token of a 1B-shaped layer joins an open block: the smallest store
        dict(name="store_1b_token", kind="store", **heads_1b, n_ctx=2304, pos=2175, t=1),
        # a whole prompt of an 8B-shaped layer
        dict(name="store_8b_prompt", kind="store", **heads_8b, n_ctx=4096, pos=0, t=2048),
        # one token late in the context of a 1B-shaped layer: latency
        dict(name="attend_1b_token", kind="attend", **heads_1b, n_ctx=2304, pos=2175, t=1),
        # one token over a long document, 8B heads
        dict(name="attend_8b_32k", kind="attend", **heads_8b, n_ctx=32768, pos=29999, t=1),
        # the longest context: the cache's bytes are all that counts
        dict(name="attend_8b_128k", kind="attend", **heads_8b, n_ctx=131072, pos=131071, t=1),
        # a few tokens checked together (speculation), neither a power of two;
        # "neox" heads in groups of seven
        dict(name="attend_few", kind="attend", n_head=28, n_kv=4, head_dim=128, neox=True,
             n_ctx=8192, pos=7001, t=5),
        # a 2048-token prompt of a 1B-shaped layer
        dict(name="attend_1b_prompt", kind="attend", **heads_1b, n_ctx=4096, pos=0, t=2048),
        # a ragged chunk that continues a conversation, 8B heads
        dict(name="attend_8b_chunk", kind="attend", **heads_8b, n_ctx=4096, pos=2901, t=777),
        # the whole decode-step call of an 8B-shaped layer
        dict(name="step_8b", kind="step", **heads_8b, n_ctx=4096, pos=3800, t=1),
        # the same of a 1B-shaped layer with a short cache: latency
        dict(name="step_1b_short", kind="step", **heads_1b, n_ctx=640, pos=99, t=1),
        # one sequence's logits: the usual window of 64 tokens, some biases and
        # a grammar that leaves few tokens
        dict(name="logits_1", kind="logits", rows=1, n=128256, last_n=64, seen=300, n_bias=40,
             mask=0.01),
        # a batch of sequences, long windows, masks that leave most tokens
        dict(name="logits_64", kind="logits", rows=64, n=128256, last_n=1024, seen=777,
             n_bias=64, mask=0.9),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["store", "attend", "step", "logits"], weights=[3, 5, 2, 2])[0]
    if kind == "logits":
        rows = _log_int(rng, 1, 64)
        last_n = _log_int(rng, 1, 2048)
        return dict(kind=kind, rows=rows, n=_log_int(rng, 1000, 128256), last_n=last_n,
                    seen=_log_int(rng, 1, 4096), n_bias=rng.choice([0, 1, _log_int(rng, 1, 300)]),
                    mask=rng.choice([0.0, 0.001, 0.5, 0.95]))
    head_dim = rng.choice([64, 64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 5, 8])
    c = dict(kind=kind, n_head=n_kv * rng.choice([1, 2, 3, 4, 4, 6, 7, 8]), n_kv=n_kv,
             head_dim=head_dim, neox=rng.random() < 0.5)
    if kind == "step" or (kind == "attend" and rng.random() < 0.4):
        n_ctx, t = _log_int(rng, 32, 65536), 1
    else:
        n_ctx = _log_int(rng, 64, 4096)
        t = _log_int(rng, 1, min(2048, n_ctx))
    # late in the context as often as anywhere
    last = n_ctx - t
    pos = last if rng.random() < 0.2 else rng.randint(last // 2 if rng.random() < 0.5 else 0, last)
    # no dearer than the prompt of 2048 tokens at 32 heads of 64 above
    while t > 1 and c["n_head"] * head_dim * t * (2 * pos + t) > 32 * 64 * 2048 * 2048:
        t = max(1, t // 2)
    return dict(c, n_ctx=n_ctx, pos=pos, t=t)


# ---- inputs --------------------------------------------------------------------

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1009 + salt)


def _rope_tables(n, n_rot):
    inv = ROPE_BASE ** (-2.0 * torch.arange(n_rot // 2, device=DEV, dtype=torch.float64) / n_rot)
    th = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    return torch.cos(th).float().contiguous(), torch.sin(th).float().contiguous()


def _cache_inputs(c, seed):
    """q [t, n_head * hd], k and v [t, n_kv * hd] of the call, and the keys
    (rotated) and values [n_kv, n, hd] that the cache holds before it.  Some
    channels of keys and values are larger than others, as in a trained
    model, and differently from token to token."""
    g = _gen(seed, 1)
    hd, n_kv, t = c["head_dim"], c["n_kv"], c["t"]
    n = c["pos"] + (t if c["kind"] == "attend" else 0)
    q = torch.randn(t, c["n_head"] * hd, generator=g, device=DEV)
    ch = torch.exp(0.6 * torch.randn(2, n_kv, 1, hd, generator=g, device=DEV))
    tok = torch.exp(0.2 * torch.randn(2, n_kv, n + t, 1, generator=g, device=DEV))
    old = []
    new = []
    for i in range(2):
        old.append(torch.randn(n_kv, n, hd, generator=g, device=DEV) * ch[i] * tok[i, :, :n])
        x = torch.randn(n_kv, t, hd, generator=g, device=DEV) * ch[i] * tok[i, :, n:]
        new.append(x.transpose(0, 1).reshape(t, n_kv * hd).contiguous())
    return q, new[0], new[1], old[0], old[1]


def _logits_inputs(c, seed):
    g = _gen(seed, 2)
    rows, n, last_n = c["rows"], c["n"], c["last_n"]
    logits = 3 * torch.randn(rows, n, generator=g, device=DEV)
    # tokens said before: some often (a power law over the vocabulary)
    u = torch.rand(rows, last_n, generator=g, device=DEV, dtype=torch.float64)
    said = (n * u ** 4).long().clamp_(0, n - 1)
    window = torch.zeros(rows, 1 + last_n, dtype=torch.int64, device=DEV)
    window[:, 0] = c["seen"]
    window[:, 1:] = said
    # each row its own: repetition 1 .. 1.3, presence 0 .. 0.8, frequency 0 .. 0.5
    span = torch.tensor([0.3, 0.8, 0.5], device=DEV, dtype=torch.float64)
    pen = torch.rand(rows, 3, generator=g, device=DEV, dtype=torch.float64) * span
    pen[:, 0] += 1.0
    bias = None
    if c["n_bias"]:
        m = c["n_bias"] * rows
        ids = torch.randint(0, n, (m,), generator=g, device=DEV)
        val = 4 * torch.randn(m, generator=g, device=DEV)
        off = torch.arange(0, m + 1, c["n_bias"], device=DEV, dtype=torch.int64)
        bias = (ids, val, off)
    allowed = None
    if c["mask"]:
        allowed = torch.rand(rows, n, generator=g, device=DEV) < c["mask"]
    return logits, window, pen, bias, allowed


def _pack(allowed):
    """One bit a token, token i in bit i % 32 of word i / 32 (int32 words)."""
    rows, n = allowed.shape
    w = -(-n // 32)
    b = torch.zeros(rows, w * 32, dtype=torch.int64, device=allowed.device)
    b[:, :n] = allowed
    v = (b.view(rows, w, 32) << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32).contiguous()


# ---- plain form ------------------------------------------------------------------

def _rotate(x, pos, cos, sin, neox):
    """x [t, heads, hd] at positions pos ..: each product and difference
    rounded to fp32."""
    t, half = x.shape[0], cos.shape[1]
    cs, sn = cos[pos:pos + t, None, :], sin[pos:pos + t, None, :]
    y = x.clone()
    if neox:
        a, b = slice(0, half), slice(half, 2 * half)
    else:
        a, b = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    x0, x1 = x[..., a], x[..., b]
    p0, p1 = x0 * cs, x1 * sn
    y[..., a] = p0 - p1
    p0, p1 = x0 * sn, x1 * cs
    y[..., b] = p0 + p1
    return y


def _code(x):
    """x [n_kv, n, hd], n a multiple of 32 -> codes (same shape), scales
    [n_kv, n / 32].  The quotient in 64 bits: 32 would move values next to a
    half from one code to the other."""
    n_kv, n, hd = x.shape
    xb = x.view(n_kv, n // BLOCK, BLOCK * hd)
    scale = (xb.abs().amax(2).double() / 127).float()
    s = torch.where(scale == 0, 1.0, scale.double())
    code = torch.round(xb.double() / s[..., None])
    return code.to(torch.int8).view(n_kv, n, hd), scale


def _pad(x):
    n = x.shape[1]
    m = -(-n // BLOCK) * BLOCK
    return torch.nn.functional.pad(x, (0, 0, 0, m - n)) if m > n else x


def _values(code, scale):
    n_kv, n, hd = code.shape
    v = code.float().view(n_kv, n // BLOCK, BLOCK, hd) * scale[:, :, None, None]
    return v.view(n_kv, n, hd)


def _attend(q, K, V, pos, n_kv):
    t, hd = q.shape[0], K.shape[2]
    n = pos + t
    G = q.shape[1] // (n_kv * hd)
    qh = q.view(t, n_kv, G, hd).permute(1, 2, 0, 3).reshape(n_kv, G * t, hd)
    z = torch.bmm(qh, K[:, :n].transpose(1, 2).contiguous()) * (1.0 / math.sqrt(hd))
    if t > 1:
        z = z.view(n_kv, G, t, n)
        see = (torch.arange(n, device=q.device)[None, :]
               <= pos + torch.arange(t, device=q.device)[:, None])
        z = z.masked_fill(~see, float("-inf")).view(n_kv, G * t, n)
    e = torch.exp(z - z.amax(2, keepdim=True))
    o = torch.bmm(e, V[:, :n].contiguous()) / e.sum(2, keepdim=True)
    return o.view(n_kv, G, t, hd).permute(2, 0, 1, 3).reshape(t, -1).contiguous()


def _plain_store(st):
    """The changed blocks coded anew from their tokens, into the state's
    cache; the rotated q and the values of the blocks up to the last token."""
    c = st["case"]
    t, n_kv, hd, pos = c["t"], c["n_kv"], c["head_dim"], c["pos"]
    q = _rotate(st["q"].view(t, -1, hd), pos, st["cos"], st["sin"], c["neox"])
    k = _rotate(st["k"].view(t, n_kv, hd), pos, st["cos"], st["sin"], c["neox"])
    v = st["v"].view(t, n_kv, hd)
    p0 = pos // BLOCK * BLOCK
    out = []
    for x, tail, (code, scale) in ((k, st["k_tail"], st["K"]), (v, st["v_tail"], st["V"])):
        blk = _pad(torch.cat([tail, x.transpose(0, 1)], dim=1))
        cd, sc = _code(blk)
        code[:, p0:p0 + cd.shape[1]] = cd
        scale[:, p0 // BLOCK:p0 // BLOCK + sc.shape[1]] = sc
        out.append(_values(cd, sc)[:, :pos + t - p0].contiguous())
    return q.view(t, -1), out[0], out[1]


def _plain_logits(st):
    x, window, pen, n = st["logits"], st["window"], st["pen"].float(), st["case"]["n"]
    last_n = window.shape[1] - 1
    cnt = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    live = torch.arange(last_n, device=x.device) < window[:, :1]
    cnt.scatter_add_(1, window[:, 1:], live.float())
    rep, pres, freq = (pen[:, i:i + 1] for i in range(3))
    said = cnt > 0
    y = torch.where(said, torch.where(x > 0, x / rep, x * rep) - pres - freq * cnt, x)
    if st["bias"] is not None:
        ids, val, off = st["bias"]
        row = torch.repeat_interleave(torch.arange(x.shape[0], device=x.device), off.diff(),
                                      output_size=ids.numel())
        last = torch.full((x.numel(),), -1, dtype=torch.int64, device=x.device)
        last.scatter_reduce_(0, row * n + ids, torch.arange(ids.numel(), device=x.device), "amax")
        last = last.view(x.shape)
        y = torch.where(last >= 0, y + val[last.clamp(min=0)], y)
    if st["mask"] is not None:
        bits = (st["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        y = torch.where(bits.view(x.shape[0], -1)[:, :n] != 0, y, float("-inf"))
    return y


# ---- prepare and run -------------------------------------------------------------

def prepare(case, seed):
    c = case
    if c["kind"] == "logits":
        logits, window, pen, bias, allowed = _logits_inputs(c, seed)
        return dict(case=c, logits=logits, window=window, pen=pen, bias=bias,
                    mask=None if allowed is None else _pack(allowed))
    q, k, v, K, V = _cache_inputs(c, seed)
    st = dict(case=c, q=q, k=k, v=v)
    if c["kind"] != "attend":
        st["cos"], st["sin"] = _rope_tables(c["n_ctx"], c["head_dim"])
    if own:
        from alpacca_amd.kvcache import QuantKVCache
        cache = QuantKVCache(c["n_kv"], c["n_ctx"], c["head_dim"])
        if K.shape[1]:
            flat = [x.transpose(0, 1).reshape(x.shape[1], -1).contiguous() for x in (K, V)]
            cache.store(flat[0], flat[1], 0)
        return dict(st, cache=cache)
    p0 = c["pos"] // BLOCK * BLOCK
    st["k_tail"], st["v_tail"] = K[:, p0:].contiguous(), V[:, p0:].contiguous()
    m = -(-c["n_ctx"] // BLOCK) * BLOCK
    for name, x in (("K", K), ("V", V)):
        code = torch.zeros(c["n_kv"], m, c["head_dim"], dtype=torch.int8, device=DEV)
        scale = torch.zeros(c["n_kv"], m // BLOCK, device=DEV)
        if x.shape[1]:
            cd, sc = _code(_pad(x))
            code[:, :cd.shape[1]] = cd
            scale[:, :sc.shape[1]] = sc
        st[name] = (code, scale)
    return st


def run(state):
    st = state
    c = st["case"]
    if own:
        return _run_own(st, c)
    if c["kind"] == "logits":
        return _plain_logits(st)
    if c["kind"] == "store":
        return _plain_store(st)
    if c["kind"] == "step":
        q, k, v = _plain_store(st)
    else:
        q, k, v = st["q"], None, None
    n = -(-(c["pos"] + c["t"]) // BLOCK) * BLOCK
    K, V = (_values(code[:, :n], scale[:, :n // BLOCK]) for code, scale in (st["K"], st["V"]))
    out = _attend(q, K, V, c["pos"], c["n_kv"])
    return (out, k, v) if c["kind"] == "step" else out


def _run_own(st, c):
    if c["kind"] == "logits":
        from alpacca_amd.logits import adjust_logits
        return adjust_logits(st["logits"], window=st["window"], penalties=st["pen"],
                             bias=st["bias"], mask=st["mask"])
    cache, pos = st["cache"], c["pos"]
    if c["kind"] == "attend":
        return cache.attend(st["q"], pos)
    start = pos // BLOCK * BLOCK
    if c["kind"] == "store":
        q = cache.store(st["k"], st["v"], pos, st["cos"], st["sin"], neox=c["neox"], q=st["q"])
        return (q, *cache.read(start, pos + c["t"]))
    out = cache.step(st["q"], st["k"], st["v"], pos, st["cos"], st["sin"], neox=c["neox"])
    return (out, *cache.read(start, pos + 1))


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "logits":
        rows, n = c["rows"], c["n"]
        b = 8 * rows * n + rows * (8 * (1 + min(c["last_n"], c["seen"])) + 24)
        b += rows * (12 * c["n_bias"] + 8) if c["n_bias"] else 0
        b += rows * 4 * -(-n // 32) if c["mask"] else 0
        return {"bytes": b, "flops": rows * (4 * min(c["last_n"], c["seen"]) + c["n_bias"])}
    hd, n_kv, n_head, t, pos = c["head_dim"], c["n_kv"], c["n_head"], c["t"], c["pos"]
    scored = t * pos + t * (t + 1) // 2  # (token, position) pairs
    att_bytes = 2 * n_kv * (pos + t) * hd + 2 * n_kv * 4 * -(-(pos + t) // BLOCK)
    att_bytes += 8 * t * n_head * hd
    att_flops = 4 * n_head * hd * scored
    if c["kind"] == "attend":
        return {"bytes": att_bytes, "flops": att_flops}
    start = pos // BLOCK * BLOCK
    # tokens in (and those of the open block before them), values of the blocks out
    b = 4 * 2 * n_kv * hd * (t + pos - start) + 4 * 2 * n_kv * hd * (pos + t - start)
    b += 2 * n_kv * hd * (pos + t - start)  # the codes
    b += 4 * t * hd  # the rows of the rotation's tables
    flops = 3 * t * (n_head + n_kv) * hd + 2 * 2 * n_kv * hd * (pos + t - start)
    if c["kind"] == "store":
        return {"bytes": b + 8 * t * n_head * hd, "flops": flops}
    return {"bytes": b + att_bytes, "flops": flops + att_flops}


# ---- from the definitions, in 64 bits ------------------------------------------------

def _exact_blocks(x):
    """x [n, hd] float64 (float32 values) of one kv head from a block's start
    on -> the values that the codes stand for."""
    out = torch.empty_like(x)
    n, hd = x.shape
    full = n // BLOCK * BLOCK
    for a, b, m in ((0, full, BLOCK), (full, n, max(1, n - full))):
        if a == b:
            continue
        y = x[a:b].reshape(-1, m * hd)
        s = (y.abs().max(dim=1, keepdim=True).values / 127).to(torch.float32).to(torch.float64)
        r = torch.where(s > 0, y / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(y))
        lo = torch.floor(r)
        up = (r - lo > 0.5) | ((r - lo == 0.5) & (torch.remainder(lo, 2) == 1))
        out[a:b] = ((lo + up.to(torch.float64)) * s).reshape(b - a, hd)
    return out


def _exact_rotated(x, pos, hd, neox):
    """x [t, heads * hd]: as complex numbers turned by the tables' angles,
    every product and sum rounded to fp32 as the operator defines it."""
    t = x.shape[0]
    cos, sin = (m[pos:pos + t, None].double() for m in _rope_tables(pos + t, hd))
    x = x.double().view(t, -1, hd)
    pairs = (x.view(t, -1, 2, hd // 2).transpose(2, 3) if neox else x.view(t, -1, hd // 2, 2))

    def r32(a):
        return a.to(torch.float32).to(torch.float64)

    re = r32(r32(pairs[..., 0] * cos) - r32(pairs[..., 1] * sin))
    im = r32(r32(pairs[..., 0] * sin) + r32(pairs[..., 1] * cos))
    y = torch.stack([re, im], dim=3)
    y = y.transpose(2, 3) if neox else y
    return y.reshape(t, -1)


def exact(case, seed):
    c = case
    if c["kind"] == "logits":
        return _exact_logits(c, seed)
    hd, n_kv, t, pos = c["head_dim"], c["n_kv"], c["t"], c["pos"]
    q, k, v, K, V = _cache_inputs(c, seed)
    q = q.double()
    start = pos // BLOCK * BLOCK
    if c["kind"] != "attend":
        q = _exact_rotated(q, pos, hd, c["neox"])
        k = _exact_rotated(k, pos, hd, c["neox"])
        K = torch.cat([K.double(), k.view(t, n_kv, hd).transpose(0, 1)], dim=1)
        V = torch.cat([V.double(), v.double().view(t, n_kv, hd).transpose(0, 1)], dim=1)
    kb, vb, outs = [], [], []
    G = c["n_head"] // n_kv
    for h in range(n_kv):
        lo = start if c["kind"] == "store" else 0
        Kh, Vh = _exact_blocks(K[h, lo:].double()), _exact_blocks(V[h, lo:].double())
        kb.append(Kh[start - lo:])
        vb.append(Vh[start - lo:])
        if c["kind"] == "store":
            continue
        for g in range(G):
            qh = q[:, (h * G + g) * hd:(h * G + g + 1) * hd]
            z = qh @ Kh.T / math.sqrt(hd)
            z += torch.full_like(z, float("-inf")).triu(pos + 1)
            outs.append(torch.softmax(z, dim=1) @ Vh)
    if c["kind"] == "attend":
        return torch.cat(outs, dim=1)
    head = q if c["kind"] == "store" else torch.cat(outs, dim=1)
    return head, torch.stack(kb), torch.stack(vb)


def _exact_logits(c, seed):
    logits, window, pen, bias, allowed = _logits_inputs(c, seed)
    y = logits.double()
    for r in range(c["rows"]):
        toks = window[r, 1:1 + min(c["seen"], c["last_n"])]
        ids, cnt = torch.unique(toks, return_counts=True)
        x = y[r, ids]
        x = torch.where(x > 0, x / pen[r, 0], x * pen[r, 0])
        y[r, ids] = x - (pen[r, 1] + pen[r, 2] * cnt.double())
        if bias is not None:
            a, b = int(bias[2][r]), int(bias[2][r + 1])
            add = dict(zip(bias[0][a:b].tolist(), bias[1][a:b].tolist()))
            ids = torch.tensor(list(add), device=DEV)
            y[r, ids] += torch.tensor(list(add.values()), device=DEV, dtype=torch.float64)
    if allowed is not None:
        y.masked_fill_(~allowed, float("-inf"))
    return y
