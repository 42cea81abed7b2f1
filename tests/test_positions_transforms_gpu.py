"""Rotary positions in calls that are more than reading and writing memory."""
import pytest
import torch

from flodl_b200 import ops

pytestmark = pytest.mark.gpu


def test_calls_that_look_at_more_than_memory():
    """Gradients of frequencies, tangents, vmap and traces go by the plain form, which knows them; so do heads too wide for a tile's angles."""
    g = torch.Generator().manual_seed(8)
    x, dx = (torch.randn(2, 5, 3, 8, generator=g).cuda() for _ in range(2))
    f = ops.rotary_frequencies(8, device="cuda")
    want = ops.rotary(x, f)
    learned = f.clone().requires_grad_()
    (slope,) = torch.autograd.grad(ops.rotary(x, learned), learned, dx)
    step = 1e-6 * torch.arange(1, 5, device="cuda", dtype=torch.float64)
    ops.set_native(False)
    try:
        moved = [ops.rotary(x.double(), f + s * step) for s in (-1, 1)]
    finally:
        ops.set_native(True)
    # fp32 sums of 240 terms of the order of one against a difference of second order: 240 * 2^-24 * 4 and 1e-12
    assert abs((slope * step).sum() - ((moved[1] - moved[0]) * dx).sum() / 2).item() < 1e-3 * (slope.abs() * step).sum().item()
    y, dy = torch.func.jvp(lambda t: ops.rotary(t, f), (x,), (dx,))
    # one rounding of each of two products and their sum on either side
    assert torch.allclose(dy, ops.rotary(dx, f), rtol=0, atol=8 * 2.0 ** -24 * dx.abs().max().item()) and torch.allclose(y, want, rtol=0, atol=8 * 2.0 ** -24 * x.abs().max().item())
    over = torch.func.vmap(lambda t: ops.qk_norm_rotary(t, freqs=f))(torch.stack((x, dx)))
    assert torch.allclose(over[1], ops.qk_norm_rotary(dx, freqs=f), rtol=0, atol=2.0 ** -20 * 3)
    traced = torch.jit.trace(lambda t: ops.rotary(t, f), (x,), check_trace=False)
    assert torch.allclose(traced(dx), ops.rotary(dx, f), rtol=0, atol=8 * 2.0 ** -24 * dx.abs().max().item())
    turned = torch.complex(x, dx).conj().imag
    assert turned.is_neg() and torch.allclose(ops.rotary(turned, f), -ops.rotary(dx, f), rtol=0, atol=8 * 2.0 ** -24 * dx.abs().max().item())
    wide = torch.randn(1, 2, 1, 16384, generator=g).cuda()
    got, f = ops.rotary(wide, ops.rotary_frequencies(16384, device="cuda")), ops.rotary_frequencies(16384)
    a = torch.arange(2).double()[:, None] * f
    lo, hi = wide[0, :, 0].cpu().double().split(8192, -1)
    assert torch.allclose(got[0, :, 0].cpu().double(), torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1), rtol=0, atol=4 * 2.0 ** -24 * 8)
