"""Rotary positions, and the RMS norm of queries and keys in the same pass (`csrc/kernels/rotary.cu`).

`x` of both operators is what attention takes: a packed projection `[B, S, 3, H, D]`, whose values come back as they were, a pair
`(q, k)` of `[B, S, H, D]` with head counts of their own, or one such tensor. The result has the same form."""
from __future__ import annotations

import math
from typing import Optional

import torch

from ..tensor import TensorError
from .core import FLAGS, _C, _launched


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0, original_length: Optional[int] = None,
                       device=None) -> torch.Tensor:
    """Radians per position of the `rotary_dim / 2` pairs of a head, `base^(-2 i / rotary_dim)`, in fp64.

    `scaling` stretches a model's positions by `factor` for contexts longer than it was trained on: `"linear"` slows every pair by it, `"base"` raises
    the base so that the slowest pair slows by it and the fastest stays, `"wavelength"` slows the pairs that turn less than once in
    `original_length` positions, leaves those that turn more than 32 times and goes over linearly between."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise TensorError(f"rotary_dim ({rotary_dim}) must be even and at least 2")
    if not (base > 0 and factor > 0):
        raise TensorError(f"base ({base}) and factor ({factor}) must be positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "base":
        if rotary_dim < 4:
            raise TensorError("scaling \"base\" needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(base) ** (-i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "wavelength":
        if original_length is None or original_length < 1:
            raise TensorError("scaling \"wavelength\" needs original_length")
        turns = original_length * f / (2 * math.pi)
        kept = ((turns - 1) / 31).clamp(0, 1)
        f = f / factor * (1 - kept) + f * kept
    elif scaling not in (None, "base"):
        raise TensorError(f"scaling must be None, \"linear\", \"base\" or \"wavelength\", not {scaling!r}")
    return f.to(device) if device is not None else f


# ------------------------------------------------------------------------------------------- arguments
def _given(x):
    """The tensors in `x`, or a TensorError."""
    given = (x,) if torch.is_tensor(x) else tuple(x) if isinstance(x, (tuple, list)) else ()
    if not given or len(given) > 2 or not all(torch.is_tensor(t) for t in given):
        raise TensorError("x must be a tensor or a pair of them")
    return given


def is_number(v) -> bool:
    """Whether it is one number, and finite."""
    try:
        return math.isfinite(v)
    except (TypeError, ValueError, RuntimeError, OverflowError):
        return False


def _parts(x):
    """The queries and keys in `x`."""
    if torch.is_tensor(x):
        return (x[:, :, 0], x[:, :, 1]) if x.dim() == 5 else (x,)
    return tuple(x)


def _check(x, freqs, positions, offset, amplitude):
    """(tensors given, positions as [B, S] int64 or None), or a TensorError."""
    given = _given(x)
    lead = given[0]
    packed = lead.dim() == 5
    if packed and (not torch.is_tensor(x) or lead.shape[2] != 3):
        raise TensorError(f"a packed projection is one tensor [B, S, 3, H, D], not {list(lead.shape)}")
    for t in given:
        if not packed and t.dim() != 4:
            raise TensorError(f"queries and keys are [B, S, H, D], not {list(t.shape)}")
        if t.shape[:2] != lead.shape[:2] or t.shape[-1] != lead.shape[-1] or t.dtype != lead.dtype or t.device != lead.device:
            raise TensorError("queries and keys must share batch, length, head dim, type and device")
        if not t.is_floating_point():
            raise TensorError(f"queries and keys must be floating point, not {t.dtype}")
    if not torch.is_tensor(freqs):
        raise TensorError(f"freqs must be a tensor (rotary_frequencies makes it), not {type(freqs).__name__}")
    if freqs.dim() != 1 or freqs.dtype != torch.float64 or freqs.device != lead.device:
        raise TensorError("freqs must be fp64 [rotary_dim / 2] on the device of the rows (rotary_frequencies makes them)")
    if 2 * freqs.numel() > lead.shape[-1]:
        raise TensorError(f"{freqs.numel()} pairs do not fit a head of {lead.shape[-1]}")
    if not is_number(amplitude):
        raise TensorError(f"amplitude ({amplitude}) must be a finite number")
    if not is_number(offset) or int(offset) != offset or not abs(offset) < 2 ** 62:
        raise TensorError(f"offset ({offset}) must be a whole number, below 2^62")
    if positions is not None:
        if not torch.is_tensor(positions):
            raise TensorError(f"positions must be a tensor, not {type(positions).__name__}")
        if positions.is_floating_point() or positions.is_complex() or positions.dtype == torch.bool:
            raise TensorError(f"positions must be whole numbers, not {positions.dtype}")
        B, S = lead.shape[:2]
        if positions.device != lead.device or positions.dim() not in (1, 2) or positions.shape[-1] != S or (positions.dim() == 2 and positions.shape[0] not in (1, B)):
            raise TensorError(f"positions must be [S] or [B, S] on the device of the rows, not {list(positions.shape)}")
        positions = positions.to(torch.int64).expand(B, S)
    return given, positions


def _native(x, freqs, positions, offset, interleaved, amplitude, norm=False, wq=None, wk=None, eps=0.0):
    """The kernel's results, or None for a call that it does not take: another device or type, or arguments that the checks explain. At any size: the
    plain form is a dozen launches."""
    pair = isinstance(x, (tuple, list))
    if pair and (len(x) not in (1, 2) or torch.is_tensor(x[0]) and x[0].dim() == 5):
        return None
    q, k = (x if len(x) == 2 else (x[0], None)) if pair else (x, None)
    if not (FLAGS.native and torch.is_tensor(q) and q.is_cuda and (k is None or torch.is_tensor(k)) and type(offset) is int):
        return None
    try:
        out = _C().turn(q, k, freqs, positions, offset, interleaved, amplitude, norm, wq, wk, eps)
    except TypeError:         # an argument that is of none of the kinds it may be: the checks say which
        return None
    if out is None:
        return None
    _launched()
    return tuple(out) if pair else out[0]


# ------------------------------------------------------------------------------------------- plain form
def _turn(x: torch.Tensor, freqs, positions, offset, interleaved, amplitude) -> torch.Tensor:
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    pos = torch.arange(x.shape[1], device=x.device)[None] if positions is None else positions
    a = (pos + offset).double()[:, :, None, None] * freqs
    cos, sin = (amplitude * a.cos()).to(wide), (amplitude * a.sin()).to(wide)
    rot = 2 * freqs.numel()
    r, rest = x[..., :rot].to(wide), x[..., rot:].to(wide)
    if interleaved:
        lo, hi = r[..., 0::2], r[..., 1::2]
        y = torch.stack((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1).flatten(-2)
    else:
        lo, hi = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _formed(x, turned):
    """Results in the form of `x`."""
    if torch.is_tensor(x):
        return torch.stack((turned[0], turned[1], x[:, :, 2]), dim=2) if x.dim() == 5 else turned[0]
    return tuple(turned)


# ------------------------------------------------------------------------------------------------ rotary
def rotary(x, freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, offset: int = 0, interleaved: bool = False, amplitude: float = 1.0):
    """Queries and keys with their positions: pair `i` of a head at position `t` turned by `t * freqs[i]` and scaled by `amplitude`.

    `positions` [S] or [B, S] (whole numbers, on the device) or 0, 1, 2, ...; `offset` is added to them. Pair `i` is the values `i` and `i + P` of the head for `P`
    frequencies, or `2 i` and `2 i + 1` with `interleaved`; what is behind the first `2 P` values stays. Angles are taken in 64 bits."""
    out = _native(x, freqs, positions, offset, interleaved, amplitude)
    if out is not None:
        return out
    _, positions = _check(x, freqs, positions, offset, amplitude)
    return _formed(x, [_turn(t, freqs, positions, offset, interleaved, amplitude).to(t.dtype) for t in _parts(x)])


# ---------------------------------------------------------------------------------------- norm and rotary
def qk_norm_rotary(x, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None,
                   positions: Optional[torch.Tensor] = None, offset: int = 0, interleaved: bool = False, amplitude: float = 1.0, eps: float = 1e-6):
    """Queries and keys normalised per head, `x / sqrt(mean(x^2) + eps) * weight` over the head's values, then turned as `rotary` does (not at all
    without `freqs`), in one pass. The weights are [D], shared by the heads; None is ones. Statistics are taken in 32 bits."""
    if freqs is None:
        freqs = torch.empty(0, dtype=torch.float64, device=_given(x)[0].device)
    out = _native(x, freqs, positions, offset, interleaved, amplitude, True, q_weight, k_weight, eps)
    if out is not None:
        return out
    given, positions = _check(x, freqs, positions, offset, amplitude)
    D = given[0].shape[-1]
    for w in (q_weight, k_weight):
        if w is not None and (not torch.is_tensor(w) or tuple(w.shape) != (D,) or w.device != given[0].device or not w.is_floating_point()):
            raise TensorError(f"weights must be [{D}] on the device of the rows")
    if k_weight is not None and len(_parts(x)) < 2:
        raise TensorError("k_weight without keys")
    if not is_number(eps) or eps < 0:
        raise TensorError(f"eps ({eps}) must not be negative")
    out = []
    for t, w in zip(_parts(x), (q_weight, k_weight)):
        n = t if t.dtype == torch.float64 else t.float()
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + eps)
        n = n if w is None else n * w.to(n.dtype)
        out.append((_turn(n, freqs, positions, offset, interleaved, amplitude) if freqs.numel() else n).to(t.dtype))
    return _formed(x, out)
