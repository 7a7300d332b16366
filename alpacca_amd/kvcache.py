"""The KV caches of one attention layer beside the fp32 one, in HBM: in 8 bits
(QuantKVCache) and, for many sequences, paged in 16 bits (PagedKVCache).

QuantKVCache: the keys and values of one sequence in 8 bits.

A quarter of the fp32 cache's bytes (the reference keeps fp32,
alpacca/model.py:368-371), and a scratch of 18, 35 or 68 MB (head_dim 64, 128,
256) that a model's layers share.  Blocks of 32 positions of one kv head share a
scale, K and V apart; attention has float32 accuracy over the coded values
(include/alpacca_amd.h, aq_kv8, has the exact rules).  A position's code depends
on the later tokens of its block too, once they are stored: a prompt's row sees
values coded with up to 31 tokens that come after it.

* ``store(k, v, pos, cos, sin, neox, q)`` - rotate and code T tokens at
  positions ``pos`` ..; returns the rotated queries, if any were given
* ``attend(q, pos)`` - causal attention of T stored tokens' queries
* ``step(q, k, v, pos, cos, sin, neox)`` - both for one token, in one call
* ``read(start, stop)`` - the values back, in fp32

Inputs are float32 tensors on the cache's device (made contiguous where they
are not); the calls only enqueue on that device's current stream.  Calls on one
cache, its construction among them, are ordered as its stores are: on one stream,
or by events.
``alpacca_amd.model.Model(..., kv_dtype="q8")`` runs its layers on these.

PagedKVCache: the keys and values of one layer for many sequences, in fp16 or
bf16, in pages that the caller hands out (include/alpacca_amd.h, aq_paged, has the
exact rules).  Sequences may share a prefix, which attention reads once for all.

* ``append(k, v, table, pos, ...)`` - rotate tokens' queries and keys and put keys
  and values into their pages
* ``attend(q, table, pos, ..., prefix=pages, start=its length)`` - attention of a
  query a row over the prefix and the row's own pages
* ``read(table, pos, ...)`` - the values back, in the cache's type
"""
from __future__ import annotations

import ctypes

from . import _lib

BLOCK = 32  # positions that share a scale
HEAD_DIMS = (64, 128, 256)
MAX_GROUP = 16  # query heads per kv head


def check_heads(n_head: int, n_kv: int, head_dim: int) -> None:
    """ValueError for heads that the 8-bit cache's attention does not take."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"the 8-bit KV cache takes head_dim {HEAD_DIMS}, got {head_dim}")
    if n_kv < 1 or n_head < 1 or n_head % n_kv or n_head // n_kv > MAX_GROUP:
        raise ValueError(f"the 8-bit KV cache takes 1 to {MAX_GROUP} query heads per kv head, "
                         f"got {n_head} for {n_kv}")


def check_paged_heads(n_head: int, n_kv: int, head_dim: int) -> None:
    """ValueError for heads that the paged cache's attention does not take."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"the paged KV cache takes head_dim {HEAD_DIMS}, got {head_dim}")
    if n_kv < 1 or n_head < 1 or n_head % n_kv or n_head // n_kv > MAX_GROUP:
        raise ValueError(f"the paged KV cache takes 1 to {MAX_GROUP} query heads per kv head, "
                         f"got {n_head} for {n_kv}")


def check_page_size(page_size: int) -> None:
    """ValueError for a number of positions that a page does not take."""
    if page_size < 32 or page_size % 32 or page_size > 65536:
        raise ValueError(f"pages hold a multiple of 32 positions up to 65536, got {page_size}")


class _Heads:
    """What the caches' calls have in common: their arguments, rows of heads of
    head_dim on the cache's device."""

    def _rows(self, x, name: str, heads=None):
        """x as a contiguous float32 [T, heads * head_dim] on the device."""
        torch = self._torch
        if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32:
            raise ValueError(f"{name} must be a float32 tensor")
        if x.device != self.device:
            raise ValueError(f"{name} is on {x.device}, the cache on {self.device}")
        dim = x.dim()
        if dim == 1:
            x = x.unsqueeze(0)
        elif dim == 3:
            if x.shape[2] != self.head_dim:
                raise ValueError(f"{name} has shape {tuple(x.shape)}, head_dim is {self.head_dim}")
            x = x.reshape(x.shape[0], x.shape[1] * x.shape[2])
        elif dim != 2:
            raise ValueError(f"{name} must be (T, heads * head_dim), got {tuple(x.shape)}")
        if heads is not None and x.shape[1] != heads * self.head_dim:
            raise ValueError(f"{name} has {x.shape[1]} values per token, expected "
                             f"{heads} x {self.head_dim}")
        x = x.contiguous()
        return x if x.data_ptr() % 16 == 0 else x.clone()  # (the kernels load 16 bytes)

    def _query_heads(self, q) -> int:
        n, rem = divmod(q.shape[1], self.head_dim)
        if rem or n == 0 or n % self.n_kv or n // self.n_kv > MAX_GROUP:
            raise ValueError(f"q has {q.shape[1]} values per token: not a multiple of "
                             f"{self.n_kv} kv heads x head_dim {self.head_dim} of at most "
                             f"{MAX_GROUP} query heads each")
        return n

    def _call(self, fn, *args):
        """fn(*args, stream) with the cache's device current."""
        cuda = self._torch.cuda
        if cuda.current_device() == self.device.index:
            _lib.check(fn(*args, _lib.current_stream(self.device.index)))
        else:
            with cuda.device(self.device):
                _lib.check(fn(*args, _lib.current_stream(self.device.index)))

    def _out(self, out, q, qc):
        if out is None:
            out = self._torch.empty_like(qc)
            return out if q.dim() == 2 else out.view(q.shape)
        if (out.dtype != self._torch.float32 or out.numel() != qc.numel()
                or out.device != self.device or not out.is_contiguous()):
            raise ValueError("out must be a contiguous float32 tensor of q's size")
        return out


class QuantKVCache(_Heads):
    """n_ctx positions of n_kv heads of head_dim, on `device` (default: the
    current one).  ValueError for an unsupported shape.  `scratch`: another
    cache whose scratch this one shares (same head_dim and device), for caches
    whose calls are ordered, like a model's layers; without it the cache makes
    its own (scratch_nbytes), which for a short context is more than the cache."""

    def __init__(self, n_kv: int, n_ctx: int, head_dim: int, device=None, scratch=None):
        import torch
        sizes = [ctypes.c_size_t() for _ in range(4)]
        _lib.check(_lib.load().aq_kv8_sizes(n_kv, head_dim, n_ctx,
                                            *[ctypes.byref(s) for s in sizes]))
        codes, scales, tail, scr = (s.value for s in sizes)
        self._lib = _lib.ensure_device()
        self._torch = torch
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise ValueError(f"the cache lives on a GPU, not {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_kv, self.n_ctx, self.head_dim = n_kv, n_ctx, head_dim
        # positions stored so far (by calls with a host position)
        self.length = 0

        def zeros(n, dtype):
            return torch.zeros(n, dtype=dtype, device=self.device)
        self.k, self.v = zeros(codes, torch.int8), zeros(codes, torch.int8)
        self.k_scale, self.v_scale = (zeros(scales // 4, torch.float32) for _ in range(2))
        self.k_tail, self.v_tail = (zeros(tail // 4, torch.float32) for _ in range(2))
        if scratch is not None:
            if scratch.head_dim != head_dim or scratch.device != self.device:
                raise ValueError("a shared scratch needs the same head_dim and device")
            self._scratch = scratch._scratch
        else:
            self._scratch = torch.empty(scr // 4, dtype=torch.float32, device=self.device)
        self._c = _lib.KV8(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                           self.v_scale.data_ptr(), self.k_tail.data_ptr(),
                           self.v_tail.data_ptr(), self._scratch.data_ptr(), n_ctx, n_kv,
                           head_dim)
        self._ref = ctypes.addressof(self._c)

    @property
    def handle(self) -> int:
        """The aq_kv8* of the C ABI (for device-resident callers)."""
        return self._ref

    def storage_nbytes(self) -> int:
        """Bytes of HBM that hold the cache's codes, scales and tails."""
        return sum(t.numel() * t.element_size()
                   for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail,
                             self.v_tail))

    def scratch_nbytes(self) -> int:
        """Bytes of the attention's scratch, which caches may share."""
        return self._scratch.numel() * self._scratch.element_size()

    def reset(self) -> None:
        """Forget what is stored."""
        self.length = 0

    # ---- arguments -----------------------------------------------------------

    def _tables(self, cos, sin, last: int):
        """n_rot and the tables' pointers; `last`: rows the call reads."""
        if cos is None and sin is None:
            return 0, None, None
        torch = self._torch
        for x, name in ((cos, "cos"), (sin, "sin")):
            if (not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.dim() != 2
                    or x.device != self.device or not x.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous float32 (positions, n_rot / 2) "
                                 f"tensor on {self.device}")
        if cos.shape != sin.shape or cos.shape[0] < last:
            raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must agree and "
                             f"reach position {last - 1}")
        return 2 * cos.shape[1], cos.data_ptr(), sin.data_ptr()

    def _span(self, pos: int, T: int, store: bool) -> None:
        if pos < 0 or pos + T > self.n_ctx:
            raise ValueError(f"positions {pos}..{pos + T - 1} outside the cache of {self.n_ctx}")
        if not store:
            if pos + T > self.length:
                raise ValueError(f"positions up to {pos + T - 1} are not all stored "
                                 f"({self.length} are)")
            return
        if pos > self.length:
            raise ValueError(f"position {pos} leaves a gap after the {self.length} stored")

    # ---- operators -----------------------------------------------------------

    def store(self, k, v, pos: int, cos=None, sin=None, neox: bool = False, q=None, q_out=None):
        """Code the T tokens k, v (T, n_kv * head_dim) at positions pos ..,
        k rotated by cos / sin (positions, n_rot / 2; None: as it is), and
        rotate q (T, n_head * head_dim) into q_out (default: a new tensor;
        may be q), which is returned.  A position at or before the last
        stored drops what followed: as if it had never been, inside the last
        block and from a multiple of 32 on; inside an earlier block what stays
        of it counts as its codes stand for it from then on."""
        torch = self._torch
        k, v = self._rows(k, "k", self.n_kv), self._rows(v, "v", self.n_kv)
        T = k.shape[0]
        if v.shape[0] != T:
            raise ValueError(f"k has {T} tokens, v {v.shape[0]}")
        n_head, qp, op = 1, None, None
        shape = None
        if q is not None:
            shape = q.shape
            q = self._rows(q, "q")
            n_head = self._query_heads(q)
            if q.shape[0] != T:
                raise ValueError(f"k has {T} tokens, q {q.shape[0]}")
            if q_out is None:
                q_out = torch.empty_like(q)
                if len(shape) != 2:
                    q_out = q_out.view(shape)
            elif (q_out.dtype != torch.float32 or q_out.numel() != q.numel()
                  or q_out.device != self.device or not q_out.is_contiguous()):
                raise ValueError("q_out must be a contiguous float32 tensor of q's size")
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        self._span(pos, T, True)
        n_rot, cp, sp = self._tables(cos, sin, pos + T)
        if T:
            self._call(self._lib.aq_rope_kv8, qp, k.data_ptr(), v.data_ptr(), op, T, n_head, n_rot,
                       1 if neox else 0, cp, sp, None, pos, self._ref)
            self.length = pos + T
        return q_out

    def attend(self, q, pos: int, out=None):
        """Attention of the queries q (T, n_head * head_dim, rotated) at
        positions pos .., each over the positions up to its own; as q."""
        qc = self._rows(q, "q")
        n_head, T = self._query_heads(qc), qc.shape[0]
        self._span(pos, T, False)
        out = self._out(out, q, qc)
        if T:
            self._call(self._lib.aq_attention_kv8, qc.data_ptr(), self._ref, T, n_head, None, pos,
                       out.data_ptr())
        return out

    def step(self, q, k, v, pos: int, cos=None, sin=None, neox: bool = False, out=None):
        """store and attend for one token, q, k and v as they are before the
        rotation: the attention output, as q."""
        qc = self._rows(q, "q")
        k, v = self._rows(k, "k", self.n_kv), self._rows(v, "v", self.n_kv)
        n_head = self._query_heads(qc)
        if not qc.shape[0] == k.shape[0] == v.shape[0] == 1:
            raise ValueError("step takes one token")
        self._span(pos, 1, True)
        n_rot, cp, sp = self._tables(cos, sin, pos + 1)
        out = self._out(out, q, qc)
        self._call(self._lib.aq_attention_rope_kv8, qc.data_ptr(), k.data_ptr(), v.data_ptr(),
                   n_head, n_rot, 1 if neox else 0, cp, sp, None, pos, self._ref, out.data_ptr())
        self.length = pos + 1
        return out

    def read(self, start: int = 0, stop: int | None = None):
        """The values of positions start .. stop - 1 (default: all stored) as
        two float32 tensors (n_kv, stop - start, head_dim)."""
        torch = self._torch
        stop = self.length if stop is None else stop
        if not 0 <= start <= stop <= self.length:
            raise ValueError(f"positions {start}..{stop - 1} of {self.length} stored")
        kv = torch.empty((2, self.n_kv, stop - start, self.head_dim), dtype=torch.float32,
                         device=self.device)
        if stop > start:
            p = kv.data_ptr()
            self._call(self._lib.aq_kv8_read, self._ref, start, stop - start, p,
                       p + 4 * self.n_kv * (stop - start) * self.head_dim)
        return kv.unbind()


class PagedKVCache(_Heads):
    """n_pages pages of page_size (a multiple of 32) positions of n_kv heads of
    head_dim in dtype (torch.float16 or torch.bfloat16), on `device` (default: the
    current one).  ValueError for an unsupported shape.

    Which pages a sequence has is the caller's: a call's ``table`` (seqs, width),
    int32, holds a row of page numbers for each sequence, in the order of its
    positions.  Where sequences share a prefix, its positions 0 .. start - 1 lie in
    pages of its own and a row's first page begins with position ``start``.  Token i
    of a call is at position pos[i] (int64) of row seq[i] (int64; None: row i).
    A token without a place (a position below 0 or below start, a row, page or
    page number out of range) is left out, as padding is: nothing is stored for it.

    The calls only enqueue on the device's current stream; those on one cache, its
    construction among them, are ordered by the caller."""

    def __init__(self, n_kv: int, n_pages: int, head_dim: int, page_size: int = 64, dtype=None,
                 device=None):
        import torch
        dtype = torch.float16 if dtype is None else dtype
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"the paged cache holds float16 or bfloat16, not {dtype}")
        check_page_size(page_size)
        for x, what in ((n_kv, "n_kv"), (n_pages, "n_pages"), (head_dim, "head_dim")):
            if not 0 < x < 2 ** 31:  # (a C integer would keep its low bits)
                raise ValueError(f"bad cache shape: {what} {x}")
        name = "F16" if dtype == torch.float16 else "BF16"
        self._c = _lib.Paged(None, None, n_pages, page_size, n_kv, head_dim,
                             _lib.DTYPE_IDS[name])
        self._ref = ctypes.addressof(self._c)
        size = ctypes.c_size_t()
        _lib.check(_lib.load().aq_paged_sizes(self._ref, ctypes.byref(size)))
        self._lib = _lib.ensure_device()
        self._torch = torch
        self.device = torch.device("cuda" if device is None else device)
        if self.device.type != "cuda":
            raise ValueError(f"the cache lives on a GPU, not {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_kv, self.n_pages, self.head_dim = n_kv, n_pages, head_dim
        self.page_size, self.dtype = page_size, dtype
        self.k, self.v = (torch.zeros(size.value // 2, dtype=dtype, device=self.device)
                          for _ in range(2))
        self._c.k, self._c.v = self.k.data_ptr(), self.v.data_ptr()

    @property
    def handle(self) -> int:
        """The aq_paged* of the C ABI (for device-resident callers)."""
        return self._ref

    def storage_nbytes(self) -> int:
        """Bytes of HBM that hold the pages."""
        return 2 * (self.k.numel() + self.v.numel())

    # ---- arguments -----------------------------------------------------------

    def _index(self, x, name: str, dtype, dim: int):
        """x as a contiguous tensor of dtype on the device."""
        if (not isinstance(x, self._torch.Tensor) or x.dtype != dtype or x.dim() != dim
                or x.device != self.device):
            have = (f"{x.dtype} {tuple(x.shape)} on {x.device}"
                    if isinstance(x, self._torch.Tensor) else type(x).__name__)
            raise ValueError(f"{name} must be {dtype} of {dim} dimension(s) on {self.device}, "
                             f"got {have}")
        return x.contiguous()

    def _places(self, table, pos, seq, start: int, n=None):
        """The checked descriptors of a call's tokens (kept alive by the caller)
        and their C arguments but start."""
        i64 = self._torch.int64
        table = self._index(table, "table", self._torch.int32, 2)
        pos = self._index(pos, "pos", i64, 1)
        if n is not None and pos.shape[0] != n:
            raise ValueError(f"{n} tokens, but pos has {pos.shape[0]}")
        if seq is not None:
            seq = self._index(seq, "seq", i64, 1)
            if seq.shape != pos.shape:
                raise ValueError(f"seq has {seq.shape[0]} tokens, pos {pos.shape[0]}")
        if not 0 <= start < 2 ** 63:
            raise ValueError(f"start {start} is below 0 or past int64")
        return (table, pos, seq), (table.data_ptr(), table.shape[0], table.shape[1],
                                   None if seq is None else seq.data_ptr(), pos.data_ptr())

    # ---- operators -----------------------------------------------------------

    def append(self, k, v, table, pos, seq=None, start: int = 0, cos=None, sin=None,
               neox: bool = False, q=None, q_out=None):
        """Put the N tokens k, v (N, n_kv * head_dim) into their places, k rotated
        by cos / sin (positions, n_rot / 2; None: as it is), and rotate q
        (N, n_head * head_dim) into q_out (default: a new tensor; may be q), which
        is returned.  A token whose position is below 0 or past the tables is left
        out, its row of q_out as it was (a new tensor's: undefined).  Two tokens in
        one place leave it undefined whose values it holds."""
        torch = self._torch
        k, v = self._rows(k, "k", self.n_kv), self._rows(v, "v", self.n_kv)
        N = k.shape[0]
        if v.shape[0] != N:
            raise ValueError(f"k has {N} tokens, v {v.shape[0]}")
        keep, place = self._places(table, pos, seq, start, N)
        n_head, qp, op = 1, None, None
        if q is not None:
            shape = q.shape
            q = self._rows(q, "q")
            n_head = self._query_heads(q)
            if q.shape[0] != N:
                raise ValueError(f"k has {N} tokens, q {q.shape[0]}")
            if q_out is None:
                q_out = torch.empty_like(q)
                if len(shape) != 2:
                    q_out = q_out.view(shape)
            elif (q_out.dtype != torch.float32 or q_out.numel() != q.numel()
                  or q_out.device != self.device or not q_out.is_contiguous()):
                raise ValueError("q_out must be a contiguous float32 tensor of q's size")
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        n_rot, cp, sp, n_pos = 0, None, None, 0
        if cos is not None or sin is not None:
            for x, name in ((cos, "cos"), (sin, "sin")):
                if (not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.dim() != 2
                        or x.device != self.device or not x.is_contiguous()):
                    raise ValueError(f"{name} must be a contiguous float32 (positions, "
                                     f"n_rot / 2) tensor on {self.device}")
            if cos.shape != sin.shape:
                raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must agree")
            n_rot, n_pos = 2 * cos.shape[1], cos.shape[0]
            cp, sp = cos.data_ptr(), sin.data_ptr()
        if N:
            self._call(self._lib.aq_rope_paged, qp, k.data_ptr(), v.data_ptr(), op, N, n_head,
                       n_rot, 1 if neox else 0, cp, sp, n_pos, *place, start, self._ref)
        return q_out

    def attend(self, q, table, pos, seq=None, start: int = 0, prefix=None, out=None):
        """Attention of the query rows q (N, n_head * head_dim, rotated), row i over
        positions 0 .. pos[i] of its sequence: those below `start` in the pages
        `prefix` (int32, all rows share them), the others in its row of the table; as
        q.  A row whose position is below 0, or that has no place to attend to,
        gives 0."""
        torch = self._torch
        qc = self._rows(q, "q")
        n_head, N = self._query_heads(qc), qc.shape[0]
        keep, place = self._places(table, pos, seq, start, N)
        pp, n_prefix = None, 0
        if prefix is not None:
            prefix = self._index(prefix, "prefix", torch.int32, 1)
            pp, n_prefix = prefix.data_ptr(), prefix.shape[0]
        if start > n_prefix * self.page_size:
            raise ValueError(f"a prefix of {n_prefix} pages of {self.page_size} holds fewer than "
                             f"{start} positions")
        out = self._out(out, q, qc)
        if N:
            size = ctypes.c_size_t()
            _lib.check(self._lib.aq_attention_paged_scratch(self._ref, N, n_head, place[2], start,
                                                            ctypes.byref(size)))
            # of this call alone: calls on other streams, and graphs, have their own
            scratch = torch.empty(size.value, dtype=torch.uint8, device=self.device)
            self._call(self._lib.aq_attention_paged, qc.data_ptr(), self._ref, N, n_head, *place,
                       pp, n_prefix, start, scratch.data_ptr(), size.value, out.data_ptr())
        return out

    def read(self, table, pos, seq=None, start: int = 0):
        """The values that the tokens' places hold, as two tensors (N, n_kv *
        head_dim) of the cache's type; 0 for a token without a place."""
        torch = self._torch
        keep, place = self._places(table, pos, seq, start)
        N, width = pos.shape[0], self.n_kv * self.head_dim
        k, v = (torch.empty((N, width), dtype=self.dtype, device=self.device) for _ in range(2))
        if N:
            self._call(self._lib.aq_paged_read, self._ref, N, *place, start, k.data_ptr(),
                       v.data_ptr())
        return k, v


__all__ = ["BLOCK", "HEAD_DIMS", "MAX_GROUP", "PagedKVCache", "QuantKVCache", "check_heads",
           "check_page_size", "check_paged_heads"]
