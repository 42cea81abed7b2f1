"""Rotary positions and normalised queries and keys on the CPU: the plain form against the definition in 64 bits, its gradients against
differences, and every refusal."""
import math

import pytest
import torch

from flodl_b200 import ops
from flodl_b200.tensor import TensorError


def turned(x, angles, interleaved):
    """Pairs of the last dimension as complex numbers times e^(i angle); angles [B or 1, S, 1, pairs]."""
    p = angles.shape[-1]
    r, rest = x[..., :2 * p], x[..., 2 * p:]
    z = torch.complex(r[..., 0::2], r[..., 1::2]) if interleaved else torch.complex(r[..., :p], r[..., p:])
    z = z * torch.exp(1j * angles)
    y = torch.stack((z.real, z.imag), -1).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((y, rest), -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(8, 8), (12, 8), (6, 2)])
def test_rotary_is_the_definition(interleaved, dim, rot):
    g = torch.Generator().manual_seed(dim + rot)
    q, k = (torch.randn(2, 5, h, dim, generator=g, dtype=torch.float64) for h in (4, 2))
    f = ops.rotary_frequencies(rot)
    pos = torch.tensor([[3, 1, 4, 1, 5], [-2, 70000, 0, 9, 2**31]])
    a = (pos + 7).double()[:, :, None, None] * f
    got = ops.rotary((q, k), f, pos, offset=7, interleaved=interleaved, amplitude=1.25)
    for t, y in zip((q, k), got):
        want = turned(t, a, interleaved)
        want[..., :rot] *= 1.25
        assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)
    # a packed projection, positions 0, 1, 2, ...: the values come back as they were
    x = torch.randn(2, 5, 3, 4, dim, generator=g, dtype=torch.float64)
    y = ops.rotary(x, f, interleaved=interleaved)
    a = torch.arange(5).double()[None, :, None, None] * f
    assert torch.equal(y[:, :, 2], x[:, :, 2]) and torch.allclose(y[:, :, 1], turned(x[:, :, 1], a, interleaved), rtol=1e-12, atol=1e-12)
    assert torch.equal(ops.rotary(x[:, :, 0], f, interleaved=interleaved), y[:, :, 0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(interleaved):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(1, 3, h, 8, generator=g, dtype=torch.float64, requires_grad=True) for h in (2, 1))
    wq, wk = (torch.randn(8, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    f = ops.rotary_frequencies(6)
    assert torch.autograd.gradcheck(lambda q, k: ops.rotary((q, k), f, interleaved=interleaved), (q, k))
    assert torch.autograd.gradcheck(lambda *t: ops.qk_norm_rotary(t[:2], *t[2:], f, offset=3, interleaved=interleaved), (q, k, wq, wk))


def test_the_norm_is_the_definition():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 3, 2, 8, generator=g, dtype=torch.float64)
    w = torch.randn(8, generator=g, dtype=torch.float64)
    y = ops.qk_norm_rotary(x, w, None, eps=1e-3)
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-3)
    assert torch.allclose(y[:, :, 0], n[:, :, 0] * w, rtol=1e-12) and torch.allclose(y[:, :, 1], n[:, :, 1], rtol=1e-12) and torch.equal(y[:, :, 2], x[:, :, 2])
    f = ops.rotary_frequencies(4)
    z = ops.qk_norm_rotary(x, w, None, f, offset=2, eps=1e-3)
    assert torch.allclose(z[:, :, 0], ops.rotary(y[:, :, 0], f, offset=2), rtol=1e-12)
    # rows of zeros have no direction: zeros, with gradients that are numbers
    x = torch.zeros(1, 1, 1, 8, requires_grad=True)
    y = ops.qk_norm_rotary(x, None, None, f)
    y.sum().backward()
    assert (y == 0).all() and torch.isfinite(x.grad).all()


def test_narrow_types_are_rounded_once():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 4, 2, 16, generator=g).bfloat16()
    f = ops.rotary_frequencies(16)
    a = (torch.arange(4) + 100000).double()[None, :, None, None] * f
    want = turned(x.double(), a, False)
    got = ops.rotary(x, f, offset=100000)
    assert got.dtype == torch.bfloat16
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -20).all()


def test_frequencies():
    f = ops.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64))
    assert torch.allclose(ops.rotary_frequencies(8, 100.0, "linear", 4.0), f / 4)
    b = ops.rotary_frequencies(8, 100.0, "base", 4.0)
    assert math.isclose(b[0], f[0]) and math.isclose(b[-1], f[-1] / 4)
    w = ops.rotary_frequencies(64, 10000.0, "wavelength", 8.0, original_length=2048)
    f = ops.rotary_frequencies(64)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(w[turns >= 32], f[turns >= 32]) and torch.equal(w[turns <= 1], f[turns <= 1] / 8)
    assert (w[1:] < w[:-1]).all()


@pytest.mark.parametrize("shape", [(0, 4, 2, 8), (2, 0, 2, 8)])
def test_empty(shape):
    x = torch.randn(shape, requires_grad=True)
    y = ops.qk_norm_rotary((x, x), None, None, ops.rotary_frequencies(8))[1]
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape


def test_refusals():
    x, f = torch.randn(2, 4, 2, 8), ops.rotary_frequencies(8)
    bad = [
        lambda: ops.rotary_frequencies(7), lambda: ops.rotary_frequencies(0), lambda: ops.rotary_frequencies(8, base=0.0),
        lambda: ops.rotary_frequencies(8, scaling="linear", factor=0.0), lambda: ops.rotary_frequencies(8, scaling="other"),
        lambda: ops.rotary_frequencies(8, scaling="wavelength"), lambda: ops.rotary_frequencies(2, scaling="base", factor=2.0),
        lambda: ops.rotary(x[0], f), lambda: ops.rotary((x, x, x), f), lambda: ops.rotary((x, x[:, :3]), f), lambda: ops.rotary((x, x.double()), f),
        lambda: ops.rotary(x.long(), f), lambda: ops.rotary(torch.randn(2, 4, 2, 2, 8), f), lambda: ops.rotary(x, f.float()),
        lambda: ops.rotary(x, ops.rotary_frequencies(10)), lambda: ops.rotary(x, f[None]), lambda: ops.rotary(x, f, torch.arange(3)),
        lambda: ops.rotary(x, f, torch.arange(4.0)), lambda: ops.rotary(x, f, torch.zeros(3, 4).long()), lambda: ops.rotary(x, f, torch.ones(4).bool()),
        lambda: ops.rotary(x, f, offset=0.5), lambda: ops.rotary(x, f, amplitude=float("nan")),
        lambda: ops.qk_norm_rotary(x, torch.ones(7)), lambda: ops.qk_norm_rotary(x, None, torch.ones(8)), lambda: ops.qk_norm_rotary(x, eps=-1.0),
        lambda: ops.qk_norm_rotary(x, torch.ones(8).long()),
    ]
    for call in bad:
        with pytest.raises(TensorError):
            call()


def test_norm_of_nothing_is_refused():
    for x in ((), [1], (None, None)):
        with pytest.raises(TensorError, match="must be a tensor or a pair"):
            ops.qk_norm_rotary(x)
        with pytest.raises(TensorError, match="must be a tensor or a pair"):
            ops.rotary(x, ops.rotary_frequencies(2))
