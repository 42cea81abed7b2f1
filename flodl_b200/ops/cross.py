"""Attention over another sequence (`csrc/kernels/cross_attn.cu`)."""
from __future__ import annotations

import math
from typing import Optional

import torch

from ..tensor import TensorError
from .core import FLAGS, _C, _launched
from .position import is_number


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(q k^T * scale + mask) v for queries [B, Sq, H, D] over keys and values [B, Sk, Hk, D] of any other length; returns [B, Sq, H, D].

    `Hk` divides `H`: query head `h` reads key head `h // (H / Hk)`, whose gradient is the sum over them. `scale` is 1 / sqrt(D) unless given. `mask` is of keys, [B, Sk],
    [1, Sk] or [B, 1, 1, Sk]: bool, True for the keys that take part, or floating point, added to the scores. A key at False or -inf is absent, whatever its key and
    value hold, and gets no gradient; a query without any key gets zeros, one whose keys' scores are all -inf gets NaN. bf16 heads of 64 and 128 on a GPU run on the kernel, at any
    size, others as plain products in 32 bits (64 for fp64). The kernel adds up before it divides, so that values beyond 2^119 / Sk overflow, and its gradients have no second derivative."""
    return attend(q, k, v, mask, scale, False)


def attend(q, k, v, mask, scale, twice: bool) -> torch.Tensor:
    """`cross_attention`; with `twice` its gradients may be differentiated again, which goes by the plain form."""
    if FLAGS.native and torch.is_tensor(q) and q.is_cuda and q.dim() == 4:
        try:
            o = _C().cross_attention(q, k, v, mask, scale if scale is not None else 1.0 / math.sqrt(q.shape[-1] or 1), twice)
        except TypeError:         # an argument that is of none of the kinds it may be: the checks say which
            o = None
        if o is not None:
            _launched()
            return o
    return _plain(q, k, v, mask, scale)


def _plain(q, k, v, mask, scale):
    if not all(torch.is_tensor(t) and t.dim() == 4 for t in (q, k, v)):
        raise TensorError("queries, keys and values are [B, S, H, D]")
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise TensorError(f"keys {list(k.shape)} and values {list(v.shape)} must be [{B}, Sk, Hk, {D}]")
    if H == 0 or Hk == 0 or H % Hk:
        raise TensorError(f"{Hk} key heads do not divide {H} query heads")
    if not q.is_floating_point() or len({(t.dtype, t.device) for t in (q, k, v)}) != 1:
        raise TensorError("queries, keys and values must be floating point, of one type and on one device")
    if D == 0:
        raise TensorError("heads of no values")
    if scale is not None and not is_number(scale):
        raise TensorError(f"scale ({scale}) must be a finite number")
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    qh = q.to(wide).transpose(1, 2).reshape(B, Hk, H // Hk * Sq, D)
    kh, vh = (t.to(wide).transpose(1, 2) for t in (k, v))
    add = alone = absent = None
    if mask is not None:
        m = mask
        if not torch.is_tensor(m):
            raise TensorError(f"mask must be a tensor, not {type(m).__name__}")
        if m.device != q.device or not (m.dtype == torch.bool or m.is_floating_point()):
            raise TensorError("mask must be bool or floating point on the device of the rows")
        if m.dim() == 4 and m.shape[1] == 1 and m.shape[2] == 1:
            m = m[:, 0, 0]
        if m.dim() != 2 or m.shape[1] != Sk or m.shape[0] not in (1, B):
            raise TensorError(f"mask must be of keys, [{B}, {Sk}], not {list(mask.shape)}")
        absent = ~m if m.dtype == torch.bool else m == float("-inf")
        if m.dtype != torch.bool and Sk > 0:
            # Relative to the row's largest, before anything is rounded to fewer bits: an addend that a row's keys share costs its scores none. Finite values stay
            # finite, and one beyond 2^100 leaves nothing of its score, as in 64 bits.
            m = m.to(torch.promote_types(m.dtype, wide))
            top = m.detach().amax(-1, keepdim=True)
            add = (m - top.masked_fill(top.isinf(), 0.0)).masked_fill(absent, 0.0).clamp(min=torch.finfo(wide).min).to(wide)[:, None, None]
            alone = (m.detach().abs() >= 2.0 ** 100)[:, None, None]
        kh, vh = (t.masked_fill(absent[:, None, :, None], 0.0) for t in (kh, vh))
    s = (qh @ kh.transpose(-1, -2)) * scale
    if add is not None:
        s = torch.where(alone, s - s.detach(), s) + add
    if absent is not None:
        s = s.masked_fill(absent[:, None, None], float("-inf"))
    if Sk == 0:
        p = s
    else:
        top = s.detach().amax(-1, keepdim=True)
        none = absent.all(-1)[:, None, None, None] if absent is not None else None      # zeros without a key; scores that are all -inf are NaN, as their softmax is
        p = torch.exp(s - (top if none is None else top.masked_fill(none, 0.0)))
        total = p.sum(-1, keepdim=True)
        p = p / (total if none is None else total.masked_fill(none, 1.0))
    return (p @ vh).reshape(B, H, Sq, D).transpose(1, 2).to(q.dtype)
