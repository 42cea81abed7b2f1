"""Rotary positions on the GPU, to the bits that fp32 has.

u = 2^-24 is half a step of fp32. sincospif is within one step of its value (CUDA's documentation), the turn by what fp32 cuts off the angle rounds once more: sine and
cosine are within 1.5 steps, 3 u |s| and 1.5 u. A product and a sum that is rounded once are u |b s| + u |y| on top."""
from decimal import Decimal, getcontext

import pytest
import torch

from flodl_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


def check(x, y, angle, slack=0.0):
    """Halves of [..., 2 P] turned by `angle` [..., P], 64 bits, known to `slack` radians."""
    a, b = x.double().chunk(2, -1)
    c, s = angle.cos(), angle.sin()
    ec, es = ((3 * t.abs()).clamp(max=1.5) * U + slack for t in (c, s))
    for got, want, other in ((y.chunk(2, -1)[0], a * c - b * s, (a.abs() * ec + b.abs() * es + U * (b * s).abs())),
                             (y.chunk(2, -1)[1], b * c + a * s, (b.abs() * ec + a.abs() * es + U * (a * s).abs()))):
        off, bound = (got.double() - want).abs(), other + U * want.abs()
        assert (off <= bound * 1.001).all(), f"{(off / bound).max().item():.3g} times the bound"


def test_fp32_has_all_its_bits():
    x = torch.randn(1, 8192, 4, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    f = ops.rotary_frequencies(64, device="cuda")
    for offset in (0, 120000):
        y = ops.rotary(x, f, offset=offset)
        # a 64-bit product of up to 2^17 radians is off by at most 2^-37
        check(x, y, (torch.arange(8192, device="cuda") + offset).double()[None, :, None, None] * f, 2.0 ** -37)


@pytest.mark.parametrize("first", [2 ** 24, 2 ** 31 - 3, 2 ** 40 + 1, -2 ** 45, 2 ** 52 - 5])
def test_a_far_position_is_as_exact_as_the_first(first):
    getcontext().prec = 60
    f = ops.rotary_frequencies(32)
    x = torch.randn(1, 4, 1, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    at = torch.tensor([first, first + 1, first + 2, first + 3])
    angle = torch.tensor([[float((Decimal(p) * Decimal(w)) % (2 * PI)) for w in f.tolist()] for p in at.tolist()], dtype=torch.float64)
    y = ops.rotary(x, f.cuda(), at.cuda())
    # the angle is known to 2^-50, and so is the reference's
    check(x, y, angle[None, :, None].cuda(), 2.0 ** -48)
    assert torch.equal(ops.rotary(x, f.cuda(), offset=first), y)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 6), (torch.bfloat16, 64), (torch.bfloat16, 10)])
def test_subnormal_values_stay(dtype, D, interleaved):
    """A turn by nothing gives back every value; others are rounded once at each product and sum, half a step of 2^-149 (2^-133 in bf16) at the least."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(1, 3, 2, D, device="cuda", generator=g) * 2.0 ** -130).to(dtype)
    assert (x != 0).any()
    f = ops.rotary_frequencies(D, device="cuda")
    y = ops.rotary(x, f, interleaved=interleaved)
    assert torch.equal(y[:, 0], x[:, 0])
    want = ops.rotary(x.double(), f, interleaved=interleaved)
    step = 2.0 ** (-149 if dtype == torch.float32 else -133)
    assert ((y.double() - want).abs() <= 2.0 ** -149 + step / 2 + 8 * U * 2.0 ** -127).all()
    (dx,) = torch.autograd.grad(ops.rotary(x.requires_grad_(), f, interleaved=interleaved), x, x.detach())
    assert torch.equal(dx[:, 0], x[:, 0])


@pytest.mark.parametrize("D", [64, 6])
def test_norms_of_subnormal_values(D):
    """x / sqrt(eps) is an ordinary value, and so is the gradient of an ordinary one: dx = w g / sqrt(eps), far from x."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(2, 3, 2, D, device="cuda", generator=g) * s for s in (2.0 ** -130, 2.0 ** -130))
    f = ops.rotary_frequencies(D, device="cuda")
    x.requires_grad_()
    y = ops.qk_norm_rotary(x, None, None, f)
    (dx,) = torch.autograd.grad(y, x, dy)
    xd = x.detach().double()
    # an fp32 eps (half a step), a reciprocal root (2 u... 4 u), a product, a turn (8 u), and subnormal steps of 2^-149 that the root raises by 1000
    for got, want in ((y, ops.rotary(xd * 1000, f)), (dx, ops.rotary(dy.double(), -f) * 1000)):
        assert ((got.double() - want).abs() <= 24 * U * 2.0 ** -117 + 2000 * 2.0 ** -149).all()
