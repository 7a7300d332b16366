"""Adjustment of logits before a token is chosen: penalties for tokens already
said, per-token biases and a grammar's mask, for the rows of a batch in one
launch (include/alpacca_amd.h, aq_logits_adjust, has the exact rules).  The
repetition penalty is the reference sampler's (alpacca/sample.py:36-45).

``Model.generate_greedy`` runs it between the head and the choice of the token.
"""
from __future__ import annotations

from . import _lib


def pack_mask(allowed):
    """A bool tensor (n,) or (rows, n) of allowed tokens as the mask's words:
    int32 (words,) or (rows, words), token t in bit t % 32 of word t // 32."""
    import torch
    if not isinstance(allowed, torch.Tensor) or allowed.dtype != torch.bool or \
            allowed.dim() not in (1, 2):
        raise ValueError("allowed must be a bool tensor (n,) or (rows, n)")
    n = allowed.shape[-1]
    w = -(-n // 32)
    bits = torch.zeros(*allowed.shape[:-1], w * 32, dtype=torch.int64, device=allowed.device)
    bits[..., :n] = allowed
    v = (bits.unflatten(-1, (w, 32)) << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)


def _tensor(x, name, dtype, shape, device):
    import torch
    if not isinstance(x, torch.Tensor) or x.dtype is not dtype or x.shape != shape:
        have = (f"{x.dtype} {tuple(x.shape)}" if isinstance(x, torch.Tensor)
                else type(x).__name__)
        raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {have}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the logits on {device}")
    return x.contiguous()


def adjust_logits(logits, *, window=None, penalties=None, bias=None, mask=None, out=None):
    """The adjusted logits (n,) or (rows, n), float32 on the GPU; `out` may be
    `logits` (default: a new tensor).  Everything else on the same device:

    window     int64 (rows, 1 + last_n): how many tokens were accepted and the
               ring of the last ones (the i-th at 1 + i % last_n)
    penalties  float64 (rows, 3): repeat, presence, frequency; with window
    bias       (ids int64, values float32), for every row, or with offsets
               int64 (rows + 1,) as a third: row r's entries are
               offsets[r] .. offsets[r + 1] - 1; a token's last entry counts
    mask       int32 words of pack_mask, (words,) for every row or
               (rows, words): tokens whose bit is clear get -inf

    (rows dropped from window and penalties for logits of one dimension.)"""
    import torch
    f32, i64 = torch.float32, torch.int64
    if not isinstance(logits, torch.Tensor) or logits.dtype != f32 or logits.dim() not in (1, 2):
        raise ValueError("logits must be a float32 tensor (n,) or (rows, n)")
    if not logits.is_cuda:
        raise ValueError("logits must be on a GPU")
    dev, one = logits.device, logits.dim() == 1
    if out is not None and not (isinstance(out, torch.Tensor) and out.dtype == f32
                                and out.shape == logits.shape and out.device == dev
                                and out.is_contiguous()):
        raise ValueError("out must be a contiguous float32 tensor of the logits' shape and device")
    x = logits.contiguous()
    rows, n = (1, x.shape[0]) if one else x.shape
    if (window is None) != (penalties is None):
        raise ValueError("window and penalties come together or not at all")
    last_n = 0
    if window is not None:
        if not isinstance(window, torch.Tensor) or window.dim() != logits.dim() \
                or window.shape[-1] < 2:
            raise ValueError("window must be int64 (rows, 1 + last_n)")
        last_n = window.shape[-1] - 1
        lead = () if one else (rows,)
        window = _tensor(window, "window", i64, (*lead, 1 + last_n), dev)
        penalties = _tensor(penalties, "penalties", torch.float64, (*lead, 3), dev)
    ids = val = off = None
    n_bias = 0
    if bias is not None:
        if not isinstance(bias, (tuple, list)) or len(bias) not in (2, 3):
            raise ValueError("bias must be (ids, values) or (ids, values, offsets)")
        n_bias = bias[0].numel() if isinstance(bias[0], torch.Tensor) else 0
        ids = _tensor(bias[0], "bias ids", i64, (n_bias,), dev)
        val = _tensor(bias[1], "bias values", f32, (n_bias,), dev)
        if len(bias) == 3:
            off = _tensor(bias[2], "bias offsets", i64, (rows + 1,), dev)
    mask_ld = 0
    if mask is not None:
        words = -(-n // 32)
        per_row = isinstance(mask, torch.Tensor) and mask.dim() == 2
        mask = _tensor(mask, "mask", torch.int32, (rows, words) if per_row else (words,), dev)
        mask_ld = words if per_row else 0
    if out is None:
        out = torch.empty_like(x)

    def p(t):
        return None if t is None else t.data_ptr()
    args = (x.data_ptr(), rows, n, p(window), last_n, p(penalties), p(ids), p(val), p(off), n_bias,
            p(mask), mask_ld, out.data_ptr())
    fn, index = _lib.ensure_device().aq_logits_adjust, dev.index
    if torch.cuda.current_device() == index:
        _lib.check(fn(*args, _lib.current_stream(index)))
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(*args, _lib.current_stream(index)))
    return out


__all__ = ["adjust_logits", "pack_mask"]
