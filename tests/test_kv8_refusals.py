"""Shapes that the 8-bit KV cache does not take are refused when a model is
built, before anything is read or moved (no GPU needed)."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")


@pytest.mark.parametrize("n_head,n_kv,head_dim", [(32, 1, 64), (34, 2, 128), (7, 2, 64),
                                                  (8, 2, 32), (8, 2, 96), (8, 2, 512), (2, 4, 64)])
def test_model_shapes(n_head, n_kv, head_dim):
    from alpacca_amd.model import Hyperparams, Model
    hp = Hyperparams("llama", 1, n_head * head_dim, n_head, n_kv, 256, 64, 64, head_dim, head_dim,
                     1e-5, 10000.0, "norm")
    with pytest.raises(ValueError, match="8-bit KV cache takes"):
        Model(hp, {}, kv_dtype="q8")


def test_heads():
    from alpacca_amd.kvcache import HEAD_DIMS, MAX_GROUP, check_heads
    for hd in HEAD_DIMS:
        check_heads(MAX_GROUP * 3, 3, hd)
        check_heads(1, 1, hd)
        with pytest.raises(ValueError):
            check_heads(MAX_GROUP * 3 + 3, 3, hd)
