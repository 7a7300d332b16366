"""The fused step on either side of the borders of its launch: one workgroup per
CU and more, a full GPU, one kv head with the most splits; the store's codes bit
for bit, and attention within the bounds of a float64 softmax."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_kv8 import dev, flat, rotate32, tables
from tests.test_kv8_long import compare, softmax64, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# 16 kv heads: 256 workgroups of five waves at 2400 positions, 272 (so four) from
# 2401 on; 512 from about 4000 on.  8: 512 from 8100 on.  1: up to 512 splits.
@pytest.mark.parametrize("hd,n_kv,G,n_ctx", [
    (64, 16, 1, 2400), (64, 16, 2, 2401), (64, 16, 1, 4100), (128, 16, 1, 2400), (128, 16, 2, 2430),
    (128, 8, 3, 8133), (64, 8, 16, 8300), (64, 1, 2, 40800), (64, 1, 2, 41000), (128, 1, 4, 70001),
    (256, 16, 1, 2400), (256, 8, 2, 4200), (256, 300, 1, 70)])
@pytest.mark.parametrize("neox", [False, True])
def test_step(hd, n_kv, G, n_ctx, neox):
    from alpacca_amd.kvcache import QuantKVCache
    n = n_ctx
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((n, n_kv, hd)).astype(np.float32) for _ in range(2))
    v += np.repeat(2 * rng.standard_normal((-(-n // 32), n_kv, hd)), 32, axis=0)[:n].astype(np.float32)
    q = rng.standard_normal((6, n_kv * G, hd)).astype(np.float32)
    cos, sin = tables(n, hd // 2)
    cd, sd, kd, vd = dev(cos), dev(sin), flat(k), flat(v)
    a = QuantKVCache(n_kv, n, hd)
    b = QuantKVCache(n_kv, n, hd, scratch=a)
    # the last positions, a block's first and last, and back into an earlier block
    at = [n - 1, (n - 1) // 32 * 32, (n - 1) // 32 * 32 - 1, n - 34, n // 2 // 32 * 32 + 5, 3]
    for i, p in enumerate(at):
        for c in (a, b):
            if i < 3:  # (stored anew: going back codes from the tail or a block's start)
                c.reset()
                c.store(kd[:p], vd[:p], 0, cd, sd, neox)
        got = a.step(flat(q[i:i + 1]), kd[p:p + 1], vd[p:p + 1], p, cd, sd, neox)
        qr = b.store(kd[p:p + 1], vd[p:p + 1], p, cd, sd, neox, q=flat(q[i:i + 1]))
        for x, y in zip(a.read(), b.read()):
            assert torch.equal(x, y), p
        if i < 3:
            K, V = values(rotate32(k[:p + 1], 0, cos, sin, neox)), values(v[:p + 1])
        else:  # (what stayed of a block is coded values, coded again)
            K, V = (x.cpu().numpy().transpose(1, 0, 2).astype(np.float64) for x in b.read())
        qr64 = rotate32(q[i:i + 1], 0, cos[p:], sin[p:], neox).astype(np.float64)
        want, tol = softmax64(qr64, K, V, p, lost=False)
        compare(got, want, tol)
        compare(b.attend(qr, p), want, tol)
