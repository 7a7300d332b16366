"""Attention and the step over long 8-bit caches: waves that take several blocks,
merges of more splits than one pass of a workgroup holds, several tiles of rows
that share the splits; against a float64 softmax over the coded values."""
from __future__ import annotations

import math

import numpy as np
import pytest

from tests.test_kv8 import B, dev, flat, rotate32, tables

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def values(x):
    """x (n, heads, hd) float32: what its codes stand for, in 64 bits."""
    n, heads, hd = x.shape
    m = -(-n // B)
    y = np.zeros((m * B, heads, hd))
    y[:n] = x
    y = y.reshape(m, B, heads, hd)
    s = (np.abs(y).max((1, 3), keepdims=True) / 127).astype(np.float32).astype(np.float64)
    return (np.rint(y / s) * s).reshape(m * B, heads, hd)[:n]


def softmax64(q, K, V, pos, lost=True):
    """q (T, n_head, hd), K / V (n, n_kv, hd): outputs and the bound of their
    error.  Scores are off by dz (products and sums as random walks of six
    standard deviations of 2^-24 of the largest sum of magnitudes, and the
    exponent's argument); weights w then by w (e^2dz - 1), and as they sum to
    one the output by that of |v - out|; sums and last roundings go by the
    largest |V|.  Asserted if `lost`: outputs without the first, a middle or the last
    whole block are out of the bound, by as much again, somewhere."""
    T, n_head, hd = q.shape
    G = n_head // K.shape[1]
    out, tol = np.empty((2, T, n_head, hd))
    for t in range(T):
        n = pos + t + 1
        for kvh in range(K.shape[1]):
            k, v, hs = K[:n, kvh], V[:n, kvh], slice(kvh * G, kvh * G + G)
            z = q[t, hs] @ k.T / math.sqrt(hd)
            mag = (np.abs(q[t, hs]) @ np.abs(k).T).max(1, keepdims=True) / math.sqrt(hd)
            top = z.max(1, keepdims=True)
            w = np.exp(z - top)
            w /= w.sum(1, keepdims=True)
            out[t, hs] = w @ v
            dz = (6 * math.sqrt(hd) * mag + np.minimum(top - z.min(1, keepdims=True), 40)) / 2 ** 24
            off = w @ np.abs(v) + np.abs(out[t, hs])  # >= w @ |v - out|
            tol[t, hs] = (np.expm1(2 * dz) * off
                          + (6 * math.sqrt(n) / 2 ** 24 + 2.0 ** -22) * np.abs(v).max())
            for b in (0, n // B // 2, n // B - 1) if lost else ():
                less = w[:, b * B:b * B + B]
                gone = less @ v[b * B:b * B + B] - less.sum(1, keepdims=True) * out[t, hs]
                assert (np.abs(gone) > 2 * tol[t, hs]).any(), (t, kvh, b)
    return out, tol


def long_inputs(n, T, n_head, n_kv, hd):
    """Keys whose scores grow over the blocks (running maxima that move) and
    values about a mean of each block's own, so that a block left out, doubled
    or taken for another one shows."""
    rng = np.random.default_rng(n + hd)
    ramp = np.repeat(np.linspace(0.4, 1.0, -(-n // B)), B)[:n, None, None]
    mean = np.repeat(3 * rng.standard_normal((-(-n // B), n_kv, hd)), B, axis=0)[:n]
    k = (rng.standard_normal((n, n_kv, hd)) * ramp).astype(np.float32)
    v = (0.5 * rng.standard_normal((n, n_kv, hd)) + mean).astype(np.float32)
    return rng.standard_normal((T, n_head, hd)).astype(np.float32), k, v


def compare(got, want, tol):
    err = np.abs(got.cpu().numpy().reshape(want.shape) - want)
    assert (err <= tol).all(), (err / tol).max()


# heads of 64, 8 kv heads: up to 256 waves per kv head, so 1 to 4 blocks each;
# one kv head: 40 splits of heads of 256 (32 in a pass), 79 of 128 (64), 313 of 64
# (more than a workgroup's threads)
@pytest.mark.parametrize("hd,n_kv,G,n,at", [(64, 8, 4, 28001, (8191, 8192, 17000, 24576, 28000)),
                                            (128, 8, 2, 20003, (8223, 16500, 20002)),
                                            (256, 1, 3, 4999, (4095, 4127, 4998)),
                                            (128, 1, 5, 10001, (8300, 10000)),
                                            (64, 1, 2, 40003, (32767, 32800, 40002)),
                                            (256, 8, 1, 20001, (20000,))])
def test_one_token(hd, n_kv, G, n, at):
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = long_inputs(n, len(at), n_kv * G, n_kv, hd)
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    K, V = values(k), values(v)
    for i, pos in enumerate(at):
        print(f"position {pos}", flush=True)
        want, tol = softmax64(q[i:i + 1].astype(np.float64), K, V, pos)
        compare(cache.attend(flat(q[i:i + 1]), pos), want, tol)


# tiles of 16 rows share the splits: 4 tiles (32 splits), 16 tiles; 64 rows a
# workgroup from 257 rows on, in 8 and fewer splits
@pytest.mark.parametrize("hd,n_kv,G,n,T", [(64, 4, 7, 9001, 9), (128, 2, 16, 12003, 16),
                                           (256, 1, 4, 6001, 17), (64, 1, 3, 9005, 90),
                                           (128, 2, 4, 8100, 70)])
def test_few_tokens(hd, n_kv, G, n, T):
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = long_inputs(n, T, n_kv * G, n_kv, hd)
    cache = QuantKVCache(n_kv, n, hd)
    cache.store(flat(k), flat(v), 0)
    want, tol = softmax64(q.astype(np.float64), values(k), values(v), n - T)
    compare(cache.attend(flat(q), n - T), want, tol)


# the step's splits take what lies before the token's block: 63 of 8 kv heads (31 of
# heads of 256), so 2 to 5 blocks per wave, and 40 / 391 of one kv head
@pytest.mark.parametrize("hd,n_kv,G,n_ctx,at,n_rot,neox", [
    (64, 8, 4, 28001, (10240, 10271, 20500, 28000), 64, False),
    (128, 8, 4, 24001, (10250, 24000), 128, True), (256, 1, 2, 4999, (4100, 4998), 64, True),
    (256, 8, 2, 20001, (16384, 20000), 0, False), (64, 1, 4, 50003, (41000, 50002), 32, False)])
def test_step(hd, n_kv, G, n_ctx, at, n_rot, neox):
    from alpacca_amd.kvcache import QuantKVCache
    q, k, v = long_inputs(n_ctx, len(at), n_kv * G, n_kv, hd)
    cos, sin = tables(n_ctx, n_rot)
    cd, sd = (dev(t) for t in (cos, sin))
    kr = rotate32(k, 0, cos, sin, neox)
    cache = QuantKVCache(n_kv, n_ctx, hd)
    kd, vd = flat(k), flat(v)
    for i, pos in enumerate(at):
        print(f"position {pos}", flush=True)
        have = cache.length
        cache.store(kd[have:pos], vd[have:pos], have, cd, sd, neox)
        got = cache.step(flat(q[i:i + 1]), kd[pos:pos + 1], vd[pos:pos + 1], pos, cd, sd, neox)
        qr = rotate32(q[i:i + 1], 0, cos[pos:], sin[pos:], neox)
        want, tol = softmax64(qr.astype(np.float64), values(kr[:pos + 1]), values(v[:pos + 1]),
                              pos)
        compare(got, want, tol)
