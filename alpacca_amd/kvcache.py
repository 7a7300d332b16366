"""QuantKVCache: the keys and values of one attention layer in 8 bits, in HBM.

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


class QuantKVCache:
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

    def _call(self, fn, *args):
        """fn(*args, stream) with the cache's device current."""
        cuda = self._torch.cuda
        if cuda.current_device() == self.device.index:
            _lib.check(fn(*args, _lib.current_stream(self.device.index)))
        else:
            with cuda.device(self.device):
                _lib.check(fn(*args, _lib.current_stream(self.device.index)))

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

    def _out(self, out, q, qc):
        if out is None:
            out = self._torch.empty_like(qc)
            return out if q.dim() == 2 else out.view(q.shape)
        if (out.dtype != self._torch.float32 or out.numel() != qc.numel()
                or out.device != self.device or not out.is_contiguous()):
            raise ValueError("out must be a contiguous float32 tensor of q's size")
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


__all__ = ["BLOCK", "HEAD_DIMS", "MAX_GROUP", "QuantKVCache", "check_heads"]
