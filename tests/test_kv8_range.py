"""Attention over the 8-bit KV cache with scores far from one: sizes of queries
and keys whose products reach 2^24 and far beyond, equal scores among them, very
small queries against very large keys and the other way round, V scales of each
block their own; every form (split, tiles, step) against a float64 softmax over
the coded values, within bounds derived below."""
from __future__ import annotations

import math

import numpy as np
import pytest

from tests.test_kv8 import B, attention64, coded, flat, inputs, values64

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def softmax_bound(q, K, V, amax, pos):
    """q (T, n_head, hd), K / V (n, n_kv, hd) float64, amax (n, n_kv) the largest
    |V| of each position's block: outputs and the bound of their error.

    Scores are off by at most dz: hd products and their sums as a random walk
    of six standard deviations, each step 2^-24 of the largest sum of
    magnitudes, and the exponent's own rounding.  Each normalised weight w then
    lies between w e^-2dz and min(1, w e^2dz), and as weights sum to one the
    output moves by at most sum |w' - w| |v - out|.  The sums' and the last
    roundings (n of 2^-24 as a random walk, 2^-22) go by the products that
    enter them."""
    T, n_head, hd = q.shape
    G = n_head // K.shape[1]
    out, tol = np.empty((2, T, n_head, hd))
    for t in range(T):
        n = pos + t + 1
        for h in range(n_head):
            k, v, am = K[:n, h // G], V[:n, h // G], amax[:n, h // G]
            z = k @ q[t, h] / math.sqrt(hd)
            logw = z - z.max() - math.log(np.exp(z - z.max()).sum())
            out[t, h] = np.exp(logw) @ v
            mag = (np.abs(k) @ np.abs(q[t, h])).max() / math.sqrt(hd)
            dz = 6 * math.sqrt(hd) * 2.0 ** -24 * mag + 2.0 ** -24 * min(z.max() - z.min(), 100)
            up, dn = np.exp(np.minimum(logw + 2 * dz, 0.0)), np.exp(logw - 2 * dz)
            tol[t, h] = ((up - dn)[:, None] * np.abs(v - out[t, h])).sum(0)
            tol[t, h] += (6 * math.sqrt(n) * 2.0 ** -24 + 2.0 ** -22) * (up * am).sum()
    return out, tol


def block_amax(v):
    """(n, n_kv): the largest magnitude of each position's block."""
    n = v.shape[0]
    m = np.stack([np.abs(v[b:b + B]).max((0, 2)) for b in range(0, n, B)])
    return np.repeat(m, B, axis=0)[:n].astype(np.float64)


def scaled_blocks(rng, v, spread):
    """v with a power of two of its own for each block, up to 2^spread either way."""
    e = np.repeat(rng.integers(-spread, spread + 1, -(-v.shape[0] // B)), B)[:v.shape[0]]
    return (v * np.exp2(e)[:, None, None]).astype(np.float32)


def compare(got, q, k, v, pos, hd):
    want, tol = softmax_bound(q.astype(np.float64), values64(*coded(k)), values64(*coded(v)),
                              block_amax(v), pos)
    got = got.cpu().numpy().reshape(want.shape).astype(np.float64)
    assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:5]
    err = np.abs(got - want)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("hd,n_kv,G", [(64, 2, 4), (128, 1, 7), (256, 1, 2)])
@pytest.mark.parametrize("size", [30.0, 300.0, 3e3, 1e4, 1e5, 1e8, 1e13, 1e18])
def test_large_scores(hd, n_kv, G, T, size):
    """q and k of this size each, so scores of about its square."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + T)
    n = 330
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    q, k = (q * np.float32(size)).astype(np.float32), (k * np.float32(size)).astype(np.float32)
    v = scaled_blocks(rng, v, 20)
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    pos = n - T
    compare(cache.attend(flat(q[pos:]), pos), q[pos:], k, v, pos, hd)


@pytest.mark.parametrize("hd,n_kv,G", [(64, 2, 4), (128, 1, 7), (256, 1, 2)])
@pytest.mark.parametrize("size", [3e3, 1e5, 1e18])
def test_large_scores_of_a_step(hd, n_kv, G, size):
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd)
    n = 200
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    q, k = (q * np.float32(size)).astype(np.float32), (k * np.float32(size)).astype(np.float32)
    v = scaled_blocks(rng, v, 20)
    cache = QuantKVCache(n_kv, n, hd)
    for p in (0, 1, 31, 32, 150, 199):
        if p > cache.length:
            cache.store(flat(k[:p]), flat(v[:p]), 0)
        got = cache.step(flat(q[p:p + 1]), flat(k[p:p + 1]), flat(v[p:p + 1]), p)
        compare(got, q[p:p + 1], k[:p + 1], v[:p + 1], p, hd)


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("size", [1.0, 300.0, 3e3, 1e4, 1e5, 1e9, 1e18])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_equal_large_scores(hd, size, T):
    """Every block holds the same keys, so the scores of a position are equal
    in every block, whatever their roundings, and whole blocks weigh alike;
    their V scales differ.  Within a block the largest score leads by far
    more than the roundings (asserted), so from size 300 on the output is the
    mean of the blocks' values at that position."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(7 * hd + T)
    nb, n_kv, G = 11, 2, 2
    n = nb * B
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    # a leading position in each block: a key along the direction that the
    # group's queries share but for a little noise; the rest small
    q = (np.repeat(q[:1, ::G], G, axis=1) + 0.01 * q).astype(np.float32)
    k = np.repeat(0.1 * k[:1], B, axis=0) * rng.uniform(0.1, 1, (B, 1, 1))
    for h in range(n_kv):
        k[5, h] = 2 * q[0, h * G]
    k = np.tile(k, (nb, 1, 1))
    q, k = ((x * size).astype(np.float32) for x in (q, k))
    v = scaled_blocks(rng, v, 12)
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    pos = n - T
    got = cache.attend(flat(q[pos:]), pos).cpu().numpy().reshape(T, n_kv * G, hd)
    K, V = values64(*coded(k)), values64(*coded(v))
    am = block_amax(v)
    for t in range(T):
        for h in range(n_kv * G):
            seen = pos + t + 1
            z = K[:B, h // G] @ q[pos + t, h].astype(np.float64) / math.sqrt(hd)  # of a block
            mag = (np.abs(K[:B, h // G]) @ np.abs(q[pos + t, h]).astype(np.float64)).max()
            dz = 6 * 2.0 ** -24 * mag + 2.0 ** -17
            zs = np.resize(z, seen)
            w = np.exp(zs - zs.max())
            top = np.sort(z)
            if size >= 300:
                assert top[-1] - top[-2] > 2 * dz + 60
                spread = 0.0  # (the others weigh nothing, the leading ones are equal)
            else:
                spread = math.expm1(2 * dz)
            w /= w.sum()
            want = w @ V[:seen, h // G]
            tol = spread * (w[:, None] * np.abs(V[:seen, h // G] - want)).sum(0)
            tol = tol + (6 * math.sqrt(seen) * 2.0 ** -24 + 2.0 ** -22) * (w * am[:seen, h // G]).sum()
            err = np.abs(got[t, h] - want)
            assert (err <= tol).all(), (t, h, (err / tol).max())


UNIT = 2.0 ** -149  # of the subnormal numbers


def of_units(u):
    """Whole units 2^-149 (magnitudes below 2^24) as float32 on the GPU, from
    their bits: a CPU that flushes subnormals does not show."""
    a = np.abs(u)
    # (below 2^24 the units are the bits: the first binade has the subnormals' unit)
    bits = (a | np.where(u < 0, 1 << 31, 0)).astype(np.uint32)
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int32)).cuda().view(torch.float32)


def test_codes_of_a_zero_scale():
    """A block whose largest magnitude is below 64 units 2^-149 has the scale
    0, and then every code is 0 and every value +0, in the store and in the
    step, also where a later token gives the block a scale."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(12)
    n_kv, hd = 2, 64
    for top in (1, 5, 63):
        u = rng.integers(-top, top + 1, (40, n_kv * hd))
        u[::B, ::hd] = -top
        x = of_units(u)
        cache = QuantKVCache(n_kv, 64, hd)
        cache.store(x, x, 0)
        q = torch.ones(1, n_kv * hd, device="cuda")
        assert (cache.attend(q, 39) == 0).all()
        for p in (None, 40):
            if p:
                cache.step(q, x[39:], x[39:], p)
            for t in (cache.k, cache.v):
                assert (t == 0).all()
            for t in (*cache.read(), cache.k_scale, cache.v_scale):
                assert (t.view(torch.int32) == 0).all()  # (no -0 either)
        cache.step(q, torch.ones_like(q), torch.ones_like(q), 41)
        for t in cache.read():
            assert (t[:, :41].view(torch.int32) & 0x7FFFFFFF == 0).all()
            assert (t[:, 41] == np.float32(1) / np.float32(127) * 127).all()


def signed(rng, lo, hi, shape):
    return rng.uniform(lo, hi, shape) * rng.choice([-1.0, 1.0], shape)


def within(got, want, tol):
    got = got.cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("hd,n_kv,G", [(64, 2, 4), (128, 1, 7), (256, 1, 2)])
@pytest.mark.parametrize("q_units,ks", [(2.0 ** 24, 1e37), (2.0 ** 22, 1e38), (2.0 ** 14, 3e38)])
def test_small_queries_and_large_keys(hd, n_kv, G, T, q_units, ks):
    """Queries of up to q_units 2^-149 (2e-38, the first two rows about the
    border of the subnormals, the last far below it), keys near the largest
    float: scores of about 1, 1 and 0.1."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + T)
    n = 230
    u = np.rint(signed(rng, 0.25 * q_units, 0.99 * q_units, (n, n_kv * G, hd))).astype(np.int64)
    k = signed(rng, 0.25 * ks, ks, (n, n_kv, hd)).astype(np.float32)
    v = signed(rng, 0.25, 1, (n, n_kv, hd)).astype(np.float32)
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    pos = n - T
    want, tol = attention64(u[pos:] * UNIT, values64(*coded(k)), values64(*coded(v)), pos)
    within(cache.attend(of_units(u[pos:].reshape(T, -1)), pos), want, tol)
    if T == 1:
        got = cache.step(of_units(u[pos:].reshape(T, -1)), flat(k[pos:]), flat(v[pos:]), pos)
        within(got, want, tol)


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("hd,n_kv,G", [(64, 2, 4), (128, 1, 7), (256, 1, 2)])
@pytest.mark.parametrize("k_units,qs", [(127.0, 3e38), (127.0 * 7, 3e38), (127.0 * 30000, 1e38)])
def test_large_queries_and_small_keys(hd, n_kv, G, T, k_units, qs):
    """Queries near the largest float, keys of up to k_units 2^-149, whose
    scales are a few units themselves."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + T)
    n = 230
    q = signed(rng, 0.25 * qs, qs, (n, n_kv * G, hd)).astype(np.float32)
    u = np.rint(signed(rng, 0.1 * k_units, k_units, (n, n_kv, hd))).astype(np.int64)
    v = signed(rng, 0.25, 1, (n, n_kv, hd)).astype(np.float32)
    s = np.stack([np.rint(np.abs(u[b:b + B]).max((0, 2)) / 127) for b in range(0, n, B)])
    s = np.repeat(s, B, axis=0)[:n, :, None]
    K = np.clip(np.rint(u / s), -127, 127) * s * UNIT
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(of_units(u.reshape(n, -1)), flat(v), 0)
    pos = n - T
    want, tol = attention64(q[pos:].astype(np.float64), K, values64(*coded(v)), pos)
    within(cache.attend(flat(q[pos:]), pos), want, tol)
    if T == 1:
        got = cache.step(flat(q[pos:]), of_units(u[pos:].reshape(1, -1)), flat(v[pos:]), pos)
        within(got, want, tol)


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("wide", [1e4, 1e7, 1e9, 1e10])
def test_queries_of_a_wide_range(hd, T, wide):
    """Two dimensions of the queries are large where every key is zero, so the
    others make the scores.  The two fp16 pieces of a row scaled to a largest
    value of 2^14 or more leave at most 2^-25 (half a unit of the second one),
    2^-39 of the row's largest magnitude; a score is off by that times the sum
    of its key's magnitudes, beside float32's own roundings."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(hd + T)
    n, n_kv, G = 230, 2, 4
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    k[..., 3] = k[..., hd // 2 + 1] = 0
    q[..., 3], q[..., hd // 2 + 1] = wide, -0.7 * wide
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    pos = n - T
    K, V = values64(*coded(k)), values64(*coded(v))
    want, tol = attention64(q[pos:].astype(np.float64), K, V, pos)
    for t in range(T):
        for h in range(n_kv * G):
            most = np.abs(K[:pos + t + 1, h // G]).sum(1).max()
            dz = 2.0 ** -39 * wide * most / math.sqrt(hd)
            tol[t, h] += 2 * np.abs(V[:pos + t + 1, h // G]).max() * math.expm1(2 * dz)
    within(cache.attend(flat(q[pos:]), pos), want, tol)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_scores_stay_finite_beside_products_past_float32(T):
    """Where every key is zero in the one dimension that holds a query's
    largest value, a block's scale times that value may pass float32: outputs
    stay means of values."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(T)
    n, n_kv, G, hd = 230, 2, 4, 64
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    k *= np.float32(1e30)
    k[..., 3] = 0
    q *= np.float32(1e-30)
    q[..., 3] = 3e38
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    V = values64(*coded(v))
    got = cache.attend(flat(q[n - T:]), n - T).cpu().numpy().reshape(T, n_kv, G, hd)
    assert np.isfinite(got).all()
    top = np.abs(V).max(0)[None, :, None] * (1 + 2.0 ** -20)
    assert (np.abs(got) <= top).all()


@pytest.mark.parametrize("T", [1, 40, 90])
@pytest.mark.parametrize("in_v", [False, True])
def test_an_infinity_reaches_its_whole_block(T, in_v):
    """Stored with the tokens of positions 64 .. 95, an infinity at 80 makes
    every row from 64 on NaN, those before it too, and no row before 64."""
    from alpacca_amd.kvcache import QuantKVCache
    rng = np.random.default_rng(T)
    n, n_kv, G, hd = 100, 2, 4, 64
    q, k, v = inputs(rng, n, n_kv * G, n_kv, hd)
    clean = values64(*coded(k)), values64(*coded(v))
    (v if in_v else k)[80, 1, 9] = -np.inf
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    for pos in sorted({0, 63 - T + 1 if T < 64 else 0, 64, n - T}):
        if pos < 0 or pos + T > n:
            continue
        want, tol = attention64(q[pos:pos + T].astype(np.float64), *clean, pos)
        got = cache.attend(flat(q[pos:pos + T]), pos).cpu().numpy().reshape(want.shape)
        for t in range(T):
            bad = slice(4, 8) if pos + t >= 64 else slice(8, 8)
            assert np.isnan(got[t, bad]).all(), (pos, t)
            good = got[t, :bad.start], want[t, :bad.start], tol[t, :bad.start]
            assert (np.abs(good[0] - good[1]) <= good[2]).all(), (pos, t)
