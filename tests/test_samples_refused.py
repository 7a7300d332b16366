"""Model.generate_samples: what one of the step's calls refuses is refused before the
model's own cache is emptied."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("kw,match", [(dict(n_seq=65536), "65535 rows"),
                                      (dict(n_seq=2 ** 31, n_gen=2), "rows"),
                                      (dict(n_seq=65536, n_gen=1), "65535 rows"),
                                      (dict(top_k=-1), "negative"),
                                      (dict(allowed=[True]), "truth values")])
def test_refused_calls_leave_the_cache(kw, match):
    from alpacca_amd.model import Model
    from tests.test_samples_model import tiny
    m = Model(*tiny())
    m.generate_greedy([1, 2, 3], 2)
    n_past, ids = m.n_past, list(m.cached_ids)
    with pytest.raises(ValueError, match=match):
        m.generate_samples(**{**dict(prompt=[1, 2], n_gen=3, n_seq=2, graph=False), **kw})
    assert m.n_past == n_past > 0 and m.cached_ids == ids
    assert len(m.generate_samples([1, 2], 3, 2)) == 2
