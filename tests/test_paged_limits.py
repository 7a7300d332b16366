"""The paged cache's calls of more rows than one launch takes (a grid holds fewer than
2^32 threads, 2^24 - 1 workgroups of 256) are refused before anything is launched; on
the CPU, where a launch would give another error."""
from __future__ import annotations

import ctypes

from alpacca_amd import _lib

P = 4096  # a pointer that nothing reads
LIMIT = 2 ** 24 - 1


def cache(n_kv, hd=64):
    return _lib.Paged(P, P, 4, 32, n_kv, hd, 1)


def append(N, n_head=4, n_kv=2, n_rot=0, neox=0, q=P):
    c = cache(n_kv)
    return _lib.load().aq_rope_paged(q, P, P, P, N, n_head, n_rot, neox, P, P, 9, P, 1, 1, None, P,
                                     0, ctypes.addressof(c), None)


def read(N, n_kv=2, hd=64):
    c = cache(n_kv, hd)
    return _lib.load().aq_paged_read(ctypes.addressof(c), N, P, 1, 1, None, P, 0, P, P, None)


def attend(N, n_head, n_kv, start=0, width=1):
    c = cache(n_kv)
    return _lib.load().aq_attention_paged(P, ctypes.addressof(c), N, n_head, P, 1, width, None, P,
                                          P, 2 ** 20, start, P, 1 << 62, P, None)


def scratch(N, n_head, n_kv, start=0, width=1):
    c, size = cache(n_kv), ctypes.c_size_t()
    rc = _lib.load().aq_attention_paged_scratch(ctypes.addressof(c), N, n_head, width, start,
                                                ctypes.byref(size))
    return rc, size.value


def test_append():
    bad = _lib.AQ_ERR_VALUE
    # a workgroup a token for queries and keys, one each four tokens for the values
    least = next(n for n in range(4 * LIMIT // 5 - 8, 2 ** 24) if n + (n + 6) // 4 > LIMIT)
    assert append(least) == bad and append(2 ** 24) == bad
    assert append(least, q=None) == bad
    assert append(2 ** 24, n_rot=20, neox=1) == bad  # in two launches: by pairs, and values
    # three workgroups a token, 68 heads of 8 threads: 3 x 5242880 + 1310721 > 2^24
    assert append(5 * 2 ** 20, n_head=64, n_kv=4) == bad


def test_read():
    assert read(2 ** 24) == _lib.AQ_ERR_VALUE
    assert read(2 ** 22, n_kv=48, hd=128) == _lib.AQ_ERR_VALUE


def test_attention():
    bad = _lib.AQ_ERR_VALUE
    # a row of a kv head a workgroup, beside those of the prefix
    assert attend(2 ** 24, 1, 1) == bad and attend(2 ** 23, 2, 2) == bad
    assert attend(LIMIT, 1, 1, start=32) == bad
    for args in ((2 ** 24, 1, 1), (2 ** 23, 2, 2), (LIMIT, 1, 1, 32)):
        assert scratch(*args)[0] == bad
    # the largest that one launch takes, however long the rows: not split past it
    assert scratch(LIMIT, 1, 1) == (_lib.AQ_OK, 0)
    assert scratch(2 ** 20, 16, 1)[0] == _lib.AQ_OK
    for n in (LIMIT, LIMIT // 2, LIMIT // 3 + 1, 2 ** 20 + 1, 700000, 3):
        for width in (1, 100, 2 ** 20, 2 ** 26 - 1):
            rc, size = scratch(n, 1, 1, width=width)
            states = max(1, size // (n * 68 * 4))  # of 64 dimensions and four numbers each
            assert rc == _lib.AQ_OK and n * states <= LIMIT, (n, width, states)


