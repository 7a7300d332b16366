"""The 8-bit KV cache (aq_rope_kv8, aq_attention_kv8, aq_attention_rope_kv8,
aq_kv8_read through alpacca_amd.kvcache): codes and scales equal to a coding in
64 bits, value for value, for every way of bringing the tokens; attention within
derived bounds of a float64 softmax over the coded values, with ragged lengths,
groups that are no power of two, rows that see one position, and infinities and
NaNs in places that a row does or does not see; refusals (on the CPU)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from alpacca_amd import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
B = 32


# ---- the definition, in 64 bits ------------------------------------------------

def rotate32(x, pos, cos, sin, neox):
    """x (T, heads, hd) float32 at positions pos ..: each product and
    difference rounded to float32."""
    T, half = x.shape[0], cos.shape[1]
    y = x.copy()
    c, s = cos[pos:pos + T, None], sin[pos:pos + T, None]
    a, b = ((slice(0, half), slice(half, 2 * half)) if neox
            else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    x0, x1 = x[..., a], x[..., b]
    y[..., a] = x0 * c - x1 * s
    y[..., b] = x0 * s + x1 * c
    return y


def coded(x):
    """x (n, heads, hd) float32 -> codes float64 (n, heads, hd), scales
    float64 (blocks, heads) of the tokens from a block's start on."""
    n, heads, hd = x.shape
    codes = np.empty((n, heads, hd))
    scales = np.empty((-(-n // B), heads))
    for b in range(scales.shape[0]):
        blk = x[b * B:(b + 1) * B].astype(np.float64)
        for h in range(heads):
            am = np.abs(blk[:, h]).max()
            if not np.isfinite(am):
                scales[b, h] = np.nan
                codes[b * B:(b + 1) * B, h] = 0
                continue
            s = np.float64(np.float32(am / 127))
            scales[b, h] = s
            codes[b * B:(b + 1) * B, h] = (np.clip(np.rint(blk[:, h] / s), -127, 127) if s > 0
                                           else 0)
    return codes, scales


def values64(codes, scales):
    return codes * np.repeat(scales, B, axis=0)[:codes.shape[0], :, None]


def attention64(q, K, V, pos):
    """q (T, n_head, hd), K / V (n, n_kv, hd) float64: outputs and bounds of
    their error relative to the largest |V| of the row's kv head: the scores'
    (HD products) and the sums' (n weights) roundings as random walks of six
    standard deviations, each step off by at most 2^-24, the exp's argument
    (2^-24 of it) and four last roundings."""
    T, n_head, hd = q.shape
    G = n_head // K.shape[1]
    out = np.empty((T, n_head, hd))
    tol = np.empty((T, n_head, 1))
    for t in range(T):
        n = pos + t + 1
        for h in range(n_head):
            k, v = K[:n, h // G], V[:n, h // G]
            z = k @ q[t, h] / math.sqrt(hd)
            w = np.exp(z - z.max())
            out[t, h] = (w @ v) / w.sum()
            mag = (np.abs(k) @ np.abs(q[t, h])).max() / math.sqrt(hd)
            dz = 6 * math.sqrt(hd) * 2.0 ** -24 * mag + 2.0 ** -24 * min(z.max() - z.min(), 40)
            tol[t, h] = np.abs(v).max() * (2 * dz + 6 * math.sqrt(n) * 2.0 ** -24 + 2.0 ** -22)
    return out, tol


def tables(n_ctx, n_rot):
    inv = 10000.0 ** (-2.0 * np.arange(n_rot // 2) / max(n_rot, 1))
    th = np.arange(n_ctx)[:, None] * inv[None]
    return np.cos(th).astype(np.float32), np.sin(th).astype(np.float32)


def inputs(rng, T, n_head, n_kv, hd):
    ch = np.exp(0.6 * rng.standard_normal((2, 1, n_kv, hd)))
    q = rng.standard_normal((T, n_head, hd)).astype(np.float32)
    k, v = ((rng.standard_normal((T, n_kv, hd)) * ch[i]).astype(np.float32) for i in range(2))
    return q, k, v


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def flat(x):
    return dev(x.reshape(x.shape[0], -1))


def same_values(cache, codes, scales, start=0):
    """The cache's values from position start (a block's first) equal s c in
    float32, bit for bit."""
    K, V = cache.read(start, start + codes[0].shape[0])
    for got, c, s in zip((K, V), codes, scales):
        want = values64(c, s).astype(np.float32).transpose(1, 0, 2)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


# ---- the store -------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("hd,n_kv,n_rot,neox,n_ctx", [(64, 8, 64, False, 200),
                                                     (128, 2, 128, True, 131),
                                                     (64, 1, 20, True, 65), (128, 3, 50, False, 97),
                                                     (256, 1, 256, False, 70), (64, 2, 0, False, 33)])
@pytest.mark.parametrize("cuts", ["one", "tokens", "ragged"])
def test_store_values(hd, n_kv, n_rot, neox, n_ctx, cuts):
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + n_ctx)
    n = n_ctx
    q, k, v = inputs(rng, n, 2 * n_kv, n_kv, hd)
    k[n // 2, 0, 3] = 1e30          # a block of large values beside ordinary ones
    v[:B, n_kv - 1] = 0             # an empty scale
    cos, sin = tables(n_ctx, n_rot)
    cache = QuantKVCache(n_kv, n_ctx, hd)
    ends = {"one": [n], "tokens": list(range(1, n + 1)),
            "ragged": sorted({1, 31, 32, 33, n // 2 + 5, n - 1, n})}[cuts]
    qd, kd, vd = flat(q), flat(k), flat(v)
    got_q = []
    a = 0
    for b in ends:
        got_q.append(cache.store(kd[a:b], vd[a:b], a, dev(cos), dev(sin), neox, q=qd[a:b]))
        a = b
    kr = rotate32(k, 0, cos, sin, neox)
    (kc, ks), (vc, vs) = coded(kr), coded(v)
    same_values(cache, (kc, vc), (ks, vs))
    want_q = rotate32(q, 0, cos, sin, neox).reshape(n, -1)
    assert np.array_equal(torch.cat(got_q).cpu().numpy(), want_q)
    assert np.array_equal(qd.cpu().numpy(), q.reshape(n, -1))  # left as it was


@gpu
def test_store_ties_and_limits():
    """Values exactly between two codes go to the even one; values next to a
    half go to their own side; the largest is 127 steps."""
    from alpacca_amd.kvcache import QuantKVCache
    hd = 64
    k = np.zeros((B, 1, hd), np.float32)
    k[0, 0, 0] = 127.0  # s = 1
    half = np.arange(-126.5, 126.6, 1.0, dtype=np.float32)
    k.reshape(-1)[1:1 + half.size] = half
    k.reshape(-1)[300:300 + half.size] = np.nextafter(half, np.float32(200))
    k.reshape(-1)[600:600 + half.size] = np.nextafter(half, np.float32(-200))
    # random scales, values within a few units of a half step of them
    rng = np.random.default_rng(3)
    v = np.empty((B, 1, hd), np.float32)
    s = np.float32(rng.uniform(0.5, 2)) * np.float32(2.0 ** -9)
    v[:] = ((rng.integers(-126, 126, v.shape) + 0.5) * np.float64(s)).astype(np.float32)
    for _ in range(3):
        step = rng.integers(-1, 2, v.shape)
        v = np.where(step > 0, np.nextafter(v, np.float32(9)),
                     np.where(step < 0, np.nextafter(v, np.float32(-9)), v)).astype(np.float32)
    v[3, 0, 5] = np.float32(127 * np.float64(s))
    cache = QuantKVCache(1, B, hd)
    cache.store(flat(k), flat(v), 0)
    (kc, ks), (vc, vs) = coded(k), coded(v)
    same_values(cache, (kc, vc), (ks, vs))
    assert kc.max() == 127


@gpu
def test_store_subnormals():
    """Values of whole units 2^-149 (expectations in whole numbers: a CPU that
    flushes subnormals does not show): the scale is the nearest unit to
    amax / 127, so a value may lie past 127 steps (and is held at 127) or the
    scale be 0 (and every code)."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(4)
    tops = np.array([5, 63, 64, 100, 189, 190, 191, 3000, 123457])
    n = tops.size * B
    u = rng.integers(-10 ** 9, 10 ** 9, (n, 64)) % (2 * np.repeat(tops, B)[:, None] + 1)
    u -= np.repeat(tops, B)[:, None]
    u[::B, 0] = tops
    bits = (np.abs(u) | np.where(u < 0, 1 << 31, 0)).astype(np.uint32)
    x = torch.from_numpy(bits.view(np.int32)).cuda().view(torch.float32)
    cache = QuantKVCache(1, n, 64)
    cache.store(x, x, 0)
    s = np.repeat(np.rint(tops / 127.0), B)[:, None]  # (no quotient is a tie)
    c = np.where(s > 0, np.clip(np.rint(u / np.maximum(s, 1)), -127, 127), 0)
    for got in cache.read():
        g = got.view(torch.int32).cpu().numpy().view(np.uint32)[0].astype(np.int64)
        g = np.where(g >> 31, -1, 1) * (g & 0x7FFFFFFF)
        assert np.array_equal(g, (c * s).astype(np.int64))


@gpu
def test_store_goes_back():
    """Back inside the last block and to the start of an earlier one: as if
    what followed had never been stored."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(5)
    _, k, v = inputs(rng, 160, 2, 2, 64)
    k[70] *= 50  # dropped below: must not leave its scale behind
    cache = QuantKVCache(2, 160, 64)
    cache.store(flat(k[:75]), flat(v[:75]), 0)
    k2, v2 = k[100:], v[100:]
    cache.store(flat(k2[:3]), flat(v2[:3]), 66)
    K, V = np.concatenate([k[:66], k2[:3]]), np.concatenate([v[:66], v2[:3]])
    (kc, ks), (vc, vs) = coded(K), coded(V)
    same_values(cache, (kc, vc), (ks, vs))
    cache.store(flat(k2[:40]), flat(v2[:40]), 32)
    K, V = np.concatenate([k[:32], k2[:40]]), np.concatenate([v[:32], v2[:40]])
    (kc, ks), (vc, vs) = coded(K), coded(V)
    same_values(cache, (kc, vc), (ks, vs))
    with pytest.raises(ValueError, match="gap"):
        cache.store(flat(k[:1]), flat(v[:1]), 80)


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("how", ["store", "step", "tokens"])
def test_store_goes_back_inside_an_earlier_block(hd, how):
    """The positions that stay of an earlier block count as their codes stand
    for them, also for tokens that join the block later."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd)
    q, k, v = inputs(rng, 160, 4, 2, hd)
    cache = QuantKVCache(2, 160, hd)
    cache.store(flat(k[:100]), flat(v[:100]), 0)
    at, n = 43, {"store": 40, "step": 1, "tokens": 5}[how]
    K, V = ([values64(*coded(x[:100])).astype(np.float32)[:at], x[100:100 + n]] for x in (k, v))
    K, V = np.concatenate(K), np.concatenate(V)
    for i, p in enumerate(range(at, at + n)) if how != "store" else ():
        if how == "step":
            cache.step(flat(q[:1]), flat(k[100:101]), flat(v[100:101]), p)
        else:
            cache.store(flat(k[100 + i:101 + i]), flat(v[100 + i:101 + i]), p)
    if how == "store":
        cache.store(flat(k[100:140]), flat(v[100:140]), at)
    # (blocks before are as they were: code them from their own tokens)
    K[:B], V[:B] = k[:B], v[:B]
    assert cache.length == at + n
    (kc, ks), (vc, vs) = coded(K), coded(V)
    same_values(cache, (kc, vc), (ks, vs))
    # the same call again on what it left
    if how == "store":
        before = [x.clone() for x in cache.read()]
        cache.store(flat(k[100:140]), flat(v[100:140]), at)
        for x, y in zip(before, cache.read()):
            assert (x - y).abs().max() <= 2.0 ** -22 * x.abs().max()


@gpu
def test_store_leaves_other_blocks_and_strided_inputs():
    """Blocks after the last stored one keep their bytes; strided and 3-D
    inputs are taken as their values."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(6)
    _, k, v = inputs(rng, 40, 2, 2, 64)
    cache = QuantKVCache(2, 128, 64)
    for t in (cache.k, cache.v):
        t.fill_(77)
    wide = torch.zeros(40, 4, 64, device="cuda")
    wide[:, ::2] = dev(k)
    cache.store(wide[:, ::2], dev(v.transpose(1, 0, 2)).transpose(0, 1), 0)
    (kc, ks), (vc, vs) = coded(k), coded(v)
    same_values(cache, (kc, vc), (ks, vs))
    for t in (cache.k, cache.v):
        assert (t.view(2, 4, B * 64)[:, 2:] == 77).all()


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_read_ranges(hd):
    """Any range of positions, from and to the middle of blocks, and nothing
    past it."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd)
    _, k, v = inputs(rng, 100, 3, 3, hd)
    cache = QuantKVCache(3, 101, hd)
    cache.store(flat(k), flat(v), 0)
    want = [values64(*coded(x)).astype(np.float32).transpose(1, 0, 2) for x in (k, v)]
    for a, b in ((0, 100), (5, 6), (31, 33), (32, 64), (40, 41), (63, 100), (99, 100), (17, 17)):
        for got, w in zip(cache.read(a, b), want):
            assert np.array_equal(got.cpu().numpy(), w[:, a:b]), (a, b)
    pad = torch.full((2, 3 * 7 * hd + 8), 9.0, device="cuda")
    _lib.check(_lib.load().aq_kv8_read(cache.handle, 29, 7, pad[0, 3:].data_ptr(),
                                       pad[1, 5:].data_ptr(), None))
    for i, off in ((0, 3), (1, 5)):
        row = pad[i].cpu().numpy()
        assert np.array_equal(row[off:off + 21 * hd], want[i][:, 29:36].reshape(-1))
        assert (row[:off] == 9).all() and (row[off + 21 * hd:] == 9).all()


@gpu
def test_store_nonfinite_blocks():
    """A block with an infinity or a NaN reads as NaN, its neighbours as
    they are; without it (gone back) the block is itself again."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(8)
    _, k, v = inputs(rng, 96, 2, 2, 64)
    k[40, 1, 7], v[95, 0, 0] = np.inf, np.nan
    cache = QuantKVCache(2, 96, 64)
    cache.store(flat(k), flat(v), 0)
    (kc, ks), (vc, vs) = coded(k), coded(v)
    assert np.isnan(ks[1, 1]) and np.isnan(vs[2, 0]) and np.isfinite(ks[1, 0])
    same_values(cache, (kc, vc), (ks, vs))
    v[95, 0, 0] = 1.0
    cache.store(flat(k[95:]), flat(v[95:]), 95)
    (vc, vs) = coded(v)
    same_values(cache, (kc, vc), (ks, vs))


# ---- attention ---------------------------------------------------------------------

def filled(rng, n_ctx, n, n_head, n_kv, hd):
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = inputs(rng, n, n_head, n_kv, hd)
    cache = QuantKVCache(n_kv, n_ctx, hd)
    cache.store(flat(k), flat(v), 0)
    return cache, q, values64(*coded(k)), values64(*coded(v))


@gpu
@pytest.mark.parametrize("hd,n_kv,G", [(64, 8, 4), (64, 1, 1), (64, 2, 7), (128, 2, 4),
                                       (128, 1, 16), (128, 3, 3), (256, 2, 2), (256, 1, 5)])
@pytest.mark.parametrize("pos", [0, 1, 30, 31, 32, 63, 64, 100, 500, 1023])
def test_attention_one_token(hd, n_kv, G, pos):
    rng = np.random.default_rng(hd + 10 * n_kv + G + pos)
    cache, q, K, V = filled(rng, max(pos + 1, 700), pos + 1, n_kv * G, n_kv, hd)
    want, tol = attention64(q[pos:].astype(np.float64), K, V, pos)
    got = cache.attend(flat(q[pos:]), pos).cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@gpu
@pytest.mark.parametrize("hd,n_kv,G,n,pos", [(64, 2, 4, 100, 0), (64, 1, 1, 130, 0),
                                             (64, 2, 8, 333, 200), (128, 2, 4, 257, 1),
                                             (128, 1, 7, 301, 129), (128, 4, 2, 96, 31),
                                             (256, 1, 4, 150, 64), (256, 2, 3, 65, 63),
                                             (64, 1, 16, 70, 5), (128, 2, 1, 1500, 1490),
                                             (64, 8, 4, 1200, 1197), (64, 4, 2, 66, 64)])
def test_attention_many_tokens(hd, n_kv, G, n, pos):
    """Chunks of n - pos tokens at pos .., from two on."""
    rng = np.random.default_rng(hd + n + pos)
    cache, q, K, V = filled(rng, n + 3, n, n_kv * G, n_kv, hd)
    want, tol = attention64(q[pos:].astype(np.float64), K, V, pos)
    got = cache.attend(flat(q[pos:]), pos).cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@gpu
@pytest.mark.parametrize("T", [1, 3, 40, 200])
@pytest.mark.parametrize("qs,ks,vs", [(1.0, 1e-30, 1e30), (1e-25, 1e25, 1e-30), (1e25, 1e-24, 1.0),
                                      (12.0, 1.0, 1.0), (1e-38, 1.0, 1.0)])
def test_attention_magnitudes(T, qs, ks, vs):
    """Far from one, and blocks of very different V scales: each row's error
    against the bound of what it sees, also where it sees the small block."""
    rng = np.random.default_rng(T)
    n, n_kv, G, hd = 230, 2, 4, 64
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    q, k, v = ((a * np.float32(s)).astype(np.float32) for a, s in ((q, qs), (k, ks), (v, vs)))
    v[-3:] *= np.float32(1e7)  # the last block's scale, seen by the last tokens alone
    cache = QuantKVCache(n_kv, n, hd)
    pos = n - T
    # token by token, so that no earlier block holds the last tokens' scale
    cache.store(flat(k), flat(v), 0)
    K, V = values64(*coded(k)), values64(*coded(v))
    want, tol = attention64(q[pos:].astype(np.float64), K, V, pos)
    got = cache.attend(flat(q[pos:]), pos).cpu().numpy().reshape(want.shape)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (err / tol).max()


@gpu
@pytest.mark.parametrize("T", [1, 2, 5, 70, 150])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_masked_nonfinite(T, hd):
    """What a row does not see does not reach it: NaN scales and codes of
    blocks past its own, whatever they hold; a block it sees makes it NaN;
    an infinity or a NaN in a query makes that row alone NaN."""
    rng = np.random.default_rng(T + hd)
    n_kv, G, n = 2, 4, 256
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    pos = 70
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k[:pos + T]), flat(v[:pos + T]), 0)
    last_blk = (pos + T - 1) // B
    for t in (cache.k_scale, cache.v_scale):  # never stored
        t.view(n_kv, -1)[:, last_blk + 1:] = float("nan")
    for t in (cache.k, cache.v):
        t.view(n_kv, -1, B * hd)[:, last_blk + 1:] = -128
    (kc, ks), (vc, vs) = coded(k[:pos + T]), coded(v[:pos + T])
    bad_from = {}
    if T >= 70:  # blocks that later rows of the call see
        for scale, blk, kvh in ((cache.k_scale, 3, 0), (cache.v_scale, 3, 1)):
            scale.view(n_kv, -1)[kvh, blk] = float("nan")
            bad_from[kvh] = blk * B
    qq = q[pos:pos + T].copy()
    if T >= 5:
        qq[3, 5, 1], qq[4, 0, 2] = np.inf, np.nan
    K, V = values64(kc, ks), values64(vc, vs)
    got = cache.attend(flat(qq), pos).cpu().numpy().reshape(T, n_kv * G, hd)
    clean = q[pos:pos + T].astype(np.float64)
    want, tol = attention64(clean, K, V, pos)
    for t in range(T):
        for h in range(n_kv * G):
            nan = not np.isfinite(qq[t, h]).all()
            nan |= h // G in bad_from and pos + t >= bad_from[h // G]
            if nan:
                assert np.isnan(got[t, h]).all(), (t, h)
            else:
                assert (np.abs(got[t, h] - want[t, h]) <= tol[t, h]).all(), (t, h)


@gpu
def test_attention_equal_keys_and_zero_query():
    """A zero query weighs all alike; a cache of zero keys and values gives
    zeros."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(2)
    cache, q, K, V = filled(rng, 100, 90, 8, 2, 64)
    for T in (1, 60):
        got = cache.attend(torch.zeros(T, 8 * 64, device="cuda"), 90 - T).cpu().numpy()
        for t in range(T):
            want = np.repeat(V[:90 - T + t + 1].mean(0), 4, axis=0)
            assert np.abs(got[t].reshape(8, 64) - want).max() < 1e-5 * np.abs(V).max()
    empty = QuantKVCache(2, 64, 64)
    z = torch.zeros(50, 128, device="cuda")
    empty.store(z, z, 0)
    assert (empty.attend(flat(q[:50]), 0) == 0).all()
    assert (empty.attend(flat(q[49:50]), 49) == 0).all()


@gpu
@pytest.mark.parametrize("hd,n_kv,G,n_rot,neox", [(64, 8, 4, 64, False), (128, 2, 7, 128, True),
                                                  (64, 2, 1, 16, True), (128, 1, 16, 34, False),
                                                  (256, 2, 2, 256, True)])
def test_step_is_store_and_attend(hd, n_kv, G, n_rot, neox):
    """The one-call step: the store's codes bit for bit, the same attention
    (within both bounds), through block borders and from the first token."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + G)
    n = 75
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    k[50] *= 30
    cos, sin = tables(n, n_rot)
    qd, kd, vd, cd, sd = flat(q), flat(k), flat(v), dev(cos), dev(sin)
    a, b = QuantKVCache(n_kv, n, hd), QuantKVCache(n_kv, n, hd)
    for p in range(n):
        step = a.step(qd[p], kd[p], vd[p], p, cd, sd, neox)
        qr = b.store(kd[p:p + 1], vd[p:p + 1], p, cd, sd, neox, q=qd[p:p + 1])
        both = b.attend(qr, p)
        for x, y in zip(a.read(), b.read()):
            assert torch.equal(x, y), p
        kr = rotate32(k[:p + 1], 0, cos, sin, neox)
        want, tol = attention64(qr.cpu().numpy().reshape(1, -1, hd).astype(np.float64),
                                values64(*coded(kr)), values64(*coded(v[:p + 1])), p)
        for got in (step, both):
            err = np.abs(got.cpu().numpy().reshape(want.shape) - want)
            assert (err <= tol).all(), (p, (err / tol).max())
    assert torch.equal(qd, flat(q)) and torch.equal(kd, flat(k))  # left as they were


@gpu
def test_state_position_capture_and_streams():
    """A position in device memory, captured once and replayed from token to
    token, with eager work between, equals the eager calls; on a stream of
    its own.  A position past the cache changes nothing."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(11)
    n_kv, G, hd, n = 2, 4, 64, 70
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    cos, sin = (dev(t) for t in tables(n, hd))
    a, b = QuantKVCache(n_kv, n, hd), QuantKVCache(n_kv, n, hd)
    lib = _lib.load()
    s = torch.cuda.Stream()
    state = torch.zeros(8, dtype=torch.int32, device="cuda")
    qs, ks, vs = (torch.zeros(m * hd, device="cuda") for m in (n_kv * G, n_kv, n_kv))
    out = torch.zeros(n_kv * G * hd, device="cuda")
    torch.cuda.synchronize()

    def call():
        _lib.check(lib.aq_attention_rope_kv8(
            qs.data_ptr(), ks.data_ptr(), vs.data_ptr(), n_kv * G, hd, 0, cos.data_ptr(),
            sin.data_ptr(), state.data_ptr(), 0, a.handle, out.data_ptr(), s.cuda_stream))
    b.step(qs, ks, vs, 0, cos, sin)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):  # nothing is allocated: no eager run of it first
        call()
    qd, kd, vd = flat(q), flat(k), flat(v)
    for p in range(n):
        with torch.cuda.stream(s):
            state[4] = p
            for dst, src in ((qs, qd), (ks, kd), (vs, vd)):
                dst.copy_(src[p])
            g.replay()
        s.synchronize()
        want = b.step(qd[p], kd[p], vd[p], p, cos, sin)
        torch.cuda.synchronize()
        assert torch.equal(out, want), p
    a.length = n
    for x, y in zip(a.read(), b.read()):
        assert torch.equal(x, y)
    before = [t.clone() for t in (a.k, a.v, a.k_scale, a.v_scale, a.k_tail, a.v_tail)]
    for p in (n, -1, 2 ** 30):
        with torch.cuda.stream(s):
            state[4] = p
            g.replay()
        s.synchronize()
        for x, y in zip(before, (a.k, a.v, a.k_scale, a.v_scale, a.k_tail, a.v_tail)):
            assert torch.equal(x, y), p


@gpu
def test_state_position_of_several_tokens():
    """aq_rope_kv8 and aq_attention_kv8 with T > 1 and the position in device
    memory: as with it on the host; tokens past the cache are skipped."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(13)
    n_kv, G, hd, n = 2, 4, 64, 90
    q, k, v = inputs(rng, n + 20, n_kv * G, n_kv, hd)
    qd, kd, vd = flat(q), flat(k), flat(v)
    a, b = QuantKVCache(n_kv, n, hd), QuantKVCache(n_kv, n, hd)
    lib = _lib.load()
    state = torch.zeros(8, dtype=torch.int32, device="cuda")
    for p, T in ((0, 37), (37, 3), (40, 1), (41, 69)):
        state[4] = p
        keep = min(T, n - p)
        out = torch.full((T, n_kv * G * hd), 5.0, device="cuda")
        _lib.check(lib.aq_rope_kv8(None, kd[p:].data_ptr(), vd[p:].data_ptr(), None, T, 1, 0, 0,
                                   None, None, state.data_ptr(), 0, a.handle, None))
        _lib.check(lib.aq_attention_kv8(qd[p:].data_ptr(), a.handle, T, n_kv * G, state.data_ptr(),
                                        0, out.data_ptr(), None))
        b.store(kd[p:p + keep], vd[p:p + keep], p)
        a.length = b.length
        for x, y in zip(a.read(), b.read()):
            assert torch.equal(x, y)
        K, V = (x.cpu().numpy().transpose(1, 0, 2).astype(np.float64) for x in b.read())
        want, tol = attention64(q[p:p + keep].astype(np.float64), K, V, p)
        got = out.cpu().numpy()
        assert (np.abs(got[:keep].reshape(want.shape) - want) <= tol).all()
        assert (got[keep:] == 5.0).all()  # rows past the cache: left as they were


# ---- refusals (no GPU needed) --------------------------------------------------------

def c_cache(n_kv=2, head_dim=64, n_ctx=100, **kw):
    p = 4096  # never followed
    c = _lib.KV8(p, p, p, p, p, p, p, n_ctx, n_kv, head_dim)
    for name, val in kw.items():
        setattr(c, name, val)
    return c


def test_sizes():
    lib = _lib.load()
    out = [ctypes.c_size_t() for _ in range(4)]
    for n_kv, hd, n_ctx in ((1, 64, 1), (8, 128, 131072), (5, 256, 33)):
        assert lib.aq_kv8_sizes(n_kv, hd, n_ctx, *map(ctypes.byref, out)) == 0
        blocks = n_kv * -(-n_ctx // B)
        assert [o.value for o in out[:3]] == [blocks * B * hd, blocks * 4,
                                              (n_kv * B * hd + -(-n_kv // 4) * 4) * 4]
        assert out[3].value > 0
    for bad in ((0, 64, 10), (1, 96, 10), (1, 64, 0), (1, 64, 2 ** 31)):
        assert lib.aq_kv8_sizes(*bad, None, None, None, None) == _lib.AQ_ERR_VALUE


def test_c_refusals():
    lib = _lib.load()
    ok = c_cache()

    def rope(c=ok, q=16, k=16, v=16, qo=16, T=1, n_head=8, n_rot=64, cos=16, sin=16, state=None,
             pos=0):
        return lib.aq_rope_kv8(q, k, v, qo, T, n_head, n_rot, 0, cos, sin, state, pos,
                               ctypes.byref(c) if c is not None else None, None)

    def attend(c=ok, q=16, T=1, n_head=8, pos=0, out=16):
        return lib.aq_attention_kv8(q, ctypes.byref(c) if c is not None else None, T, n_head, None,
                                    pos, out, None)

    def step(c=ok, q=16, k=16, v=16, n_head=8, n_rot=64, neox=0, cos=16, pos=0, out=16):
        return lib.aq_attention_rope_kv8(q, k, v, n_head, n_rot, neox, cos, 16, None, pos,
                                         ctypes.byref(c), out, None)

    def read(c=ok, start=0, n=1, k=16, v=16):
        return lib.aq_kv8_read(ctypes.byref(c), start, n, k, v, None)

    bad = [rope(c=None), attend(c=None), rope(T=-1), attend(T=-1), rope(k=None), rope(v=None),
           rope(qo=None), rope(pos=-1), rope(pos=100), rope(pos=99, T=2), rope(n_rot=3),
           rope(n_rot=66), rope(n_rot=-2), rope(cos=None), rope(n_head=0), rope(T=101),
           rope(pos=2 ** 62), rope(T=2 ** 62),
           attend(q=None), attend(out=None), attend(n_head=7), attend(n_head=0),
           attend(n_head=34), attend(T=65536, c=c_cache(n_ctx=10 ** 6)), attend(pos=100),
           attend(pos=-1), attend(T=2 ** 62),
           step(q=None), step(k=None), step(v=None), step(out=None), step(n_rot=4, neox=1),
           step(cos=None), step(pos=100), step(n_head=3),
           read(start=-1), read(start=100), read(n=101), read(n=-1), read(k=None), read(v=None),
           read(n=2 ** 62)]
    for c in (c_cache(n_kv=0), c_cache(head_dim=96), c_cache(n_ctx=0), c_cache(n_ctx=2 ** 31),
              c_cache(k=None), c_cache(v_tail=None), c_cache(v=4100), c_cache(k_tail=4100),
              c_cache(scratch=None), c_cache(scratch=4100), c_cache(k_scale=None)):
        bad += [rope(c=c), attend(c=c), step(c=c), read(c=c)]
    assert all(rc == _lib.AQ_ERR_VALUE for rc in bad), bad
    # nothing to do: no launch, so no device is needed
    assert rope(T=0) == attend(T=0) == read(n=0) == _lib.AQ_OK


@gpu
def test_python_refusals():
    from alpacca_amd.kvcache import QuantKVCache
    with pytest.raises(ValueError):
        QuantKVCache(2, 100, 96)
    with pytest.raises(ValueError):
        QuantKVCache(2, 0, 64)
    c = QuantKVCache(2, 100, 64)
    x = torch.zeros(4, 128, device="cuda")
    q = torch.zeros(4, 512, device="cuda")
    cos = torch.zeros(100, 32, device="cuda")
    for bad in (lambda: c.store(x.cpu(), x, 0), lambda: c.store(x.half(), x, 0),
                lambda: c.store(x[:, :64], x, 0), lambda: c.store(x, x[:3], 0),
                lambda: c.store(x, x, 1), lambda: c.store(x, x, -1), lambda: c.store(x, x, 98),
                lambda: c.store(x, x, 0, cos[:3], cos[:3]), lambda: c.store(x, x, 0, cos, None),
                lambda: c.store(x, x, 0, q=q[:, :192]), lambda: c.store(x, x, 0, q=q[:3]),
                lambda: c.store(x, x, 0, q_out=q), lambda: c.attend(q, 0),
                lambda: c.step(q, x, x, 0), lambda: c.read(0, 1),
                lambda: QuantKVCache(2, 100, 128, scratch=c)):
        with pytest.raises(ValueError):
            bad()
    assert c.length == 0
    assert c.store(x[:0], x[:0], 0, q=q[:0]).shape == (0, 512)
    c.store(x, x, 0)
    assert c.attend(q[:0], 4).shape == (0, 512)
