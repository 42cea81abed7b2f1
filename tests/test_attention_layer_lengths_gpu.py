"""`nn.MultiheadAttention` over keys of another length answers on the kernel what it answers as separate operators: gradients that are differentiated again, batches of
gradients, queries whose keys are all masked."""
import pytest
import torch

from flodl_b200 import nn, ops
from flodl_b200.autograd import Variable

pytestmark = pytest.mark.gpu

E, HEADS = 128, 2


def layer():
    torch.manual_seed(2)
    m = nn.MultiheadAttention(E, HEADS, "cuda")
    q, s = (torch.randn(3, n, E, device="cuda").bfloat16().requires_grad_() for n in (5, 70))
    mask = (torch.rand(3, 1, 1, 70, device="cuda") < 0.3).float()
    return m, q, s, mask


def call(m, q, s, mask, kernel=True):
    """Small projections are left to PyTorch, attention is not; or all of it to PyTorch, in the inputs' type."""
    w = Variable.wrap
    if not kernel:
        ops.set_native(False)
        try:
            return m.forward_ext(w(q), w(s), w(s), mask).t
        finally:
            ops.set_native(True)
    ops.FLAGS.count_launches, ops.FLAGS.launches = True, 0
    with nn.AutocastGuard(torch.bfloat16):
        o = m.forward_ext(w(q), w(s), w(s), mask).t
    ops.FLAGS.count_launches = False
    assert ops.FLAGS.launches == 1
    return o


def wide(m, *ts):
    for pair in m.proj.values():
        for p in pair:
            p.t.data = p.t.data.double()
    return [t.detach().double().requires_grad_() for t in ts]


@pytest.mark.parametrize("masked", [False, True])
def test_gradients_are_differentiated_again(masked):
    """Against 64 bits, relative to the largest: three chained products forth and back of bf16 roundings, 2^-8 each, some ten of them."""
    m, q, s, mask = layer()
    mask = mask if masked else None

    def second(q, s, o):
        g = torch.autograd.grad(o.square().sum(), (q, s), create_graph=True)
        return (*g, *torch.autograd.grad(sum(t.square().sum() for t in g), (q, s)))
    got = second(q, s, call(m, q, s, mask))
    qw, sw = wide(m, q, s)
    want = second(qw, sw, call(m, qw, sw, mask, kernel=False))
    for a, b in zip(got, want):
        assert a.shape == b.shape and (a.double() - b).norm() <= 10 * 2.0 ** -8 * b.norm()


def test_a_batch_of_gradients():
    m, q, s, mask = layer()
    do = torch.randn(4, 3, 5, E, device="cuda").bfloat16()
    o = call(m, q, s, mask)
    got = torch.autograd.grad(o, (q, s), do, is_grads_batched=True, retain_graph=True)
    for i in range(4):
        for a, b in zip(got, torch.autograd.grad(o, (q, s), do[i], retain_graph=True)):
            # the kernel's roundings of P and dS on one side, the projections' on both
            assert (a[i].double() - b.double()).norm() <= 4 * 2.0 ** -8 * b.double().norm()


def test_queries_without_a_key_are_as_in_separate_operators():
    m, q, s, mask = layer()
    mask[1] = 1
    o = call(m, q, s, mask)
    (dw,) = torch.autograd.grad(o.sum(), m.proj["v_proj"][0].t)
    qw, sw = wide(m, q, s)
    want = call(m, qw, sw, mask, kernel=False)
    assert torch.equal(o.isnan(), want.isnan()) and o[1].isnan().all() and not o[[0, 2]].isnan().any()
    assert dw.isnan().all()
    # one mask for the batch
    assert call(m, q, s, torch.ones(1, 70, device="cuda")).isnan().all()


def test_the_operator_itself_refuses_a_second_derivative():
    q, k = (torch.randn(1, n, 2, 64, device="cuda").bfloat16().requires_grad_() for n in (3, 9))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.cross_attention(q, k, k).sum(), q, create_graph=True)
