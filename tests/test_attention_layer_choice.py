"""Which way `nn.MultiheadAttention` goes over keys of another length: by sizes alone, and with the same result."""
import pytest
import torch

from flodl_b200 import nn, ops
from flodl_b200.autograd import Variable

# B, H, Sq, Sk, trained, masked
FASTER = [(2, 2, 5, 9, True, True), (16, 8, 1, 500, False, True), (16, 8, 1, 500, True, True), (1024, 8, 48, 200, True, True), (4096, 2, 32, 64, True, True), (8000, 2, 4, 33, False, True),
          (64, 8, 128, 256, True, False), (1, 1, 600, 3000, True, False), (409, 1, 16, 8, False, True), (930, 8, 21, 2, False, False)]
NOT = [(1412, 16, 2, 1, True, True), (2848, 16, 42, 2, True, False), (2171, 16, 64, 2, True, True), (1140, 1, 25, 112, True, True), (930, 8, 21, 2, False, True), (409, 1, 240, 1, False, True),
       (1237, 1, 89, 20, False, False)]


@pytest.mark.parametrize("sizes,kernel", [(s, True) for s in FASTER] + [(s, False) for s in NOT], ids=str)
def test_the_rule(sizes, kernel):
    assert nn.MultiheadAttention._kernel_is_faster(*sizes) == kernel


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Sq,Sk,kernel", [(400, 2, 6, 4, False), (400, 2, 40, 60, True), (90, 2, 6, 4, True)])
def test_either_way_is_the_same_layer(monkeypatch, B, H, Sq, Sk, kernel):
    monkeypatch.setitem(ops.core._EAGER, "min_numel", 1 << 40)          # projections are PyTorch's
    torch.manual_seed(3)
    m = nn.MultiheadAttention(64 * H, H, "cuda")
    q, s = (torch.randn(B, n, 64 * H, device="cuda").bfloat16().requires_grad_() for n in (Sq, Sk))
    mask = (torch.rand(B, 1, 1, Sk, device="cuda") < 0.3).float()
    mask[:, ..., 0] = 0
    mask[3] = 1
    do = torch.randn(B, Sq, 64 * H, device="cuda").bfloat16()

    def grads(dtype):
        x = [t.detach().to(dtype).requires_grad_() for t in (q, s)]
        if dtype == torch.bfloat16:
            with nn.AutocastGuard(torch.bfloat16):
                o = m.forward_ext(*(Variable.wrap(t) for t in (x[0], x[1], x[1])), mask).t
        else:
            o = m.forward_ext(*(Variable.wrap(t) for t in (x[0], x[1], x[1])), mask).t
        return (o, *torch.autograd.grad(o, x, do.to(dtype)))
    ops.FLAGS.count_launches, ops.FLAGS.launches = True, 0
    got = grads(torch.bfloat16)
    ops.FLAGS.count_launches = False
    assert ops.FLAGS.launches == (1 if kernel else 0)
    for pair in m.proj.values():
        for p in pair:
            p.t.data = p.t.data.double()
    for a, b in zip(got, grads(torch.float64)):
        assert torch.equal(a.isnan(), b.isnan()) and a[3].isnan().all()
        a, b = (t.double().nan_to_num(0.0) for t in (a, b))
        # six bf16 roundings in a row, of weights, projections, scores or P, sums, the result
        assert (a - b).norm() <= 6 * 2.0 ** -8 * b.norm()
