"""Attention over another sequence on the CPU: the plain form against the definition in 64 bits, its gradients against differences, every refusal, and the module that uses it."""
import math

import pytest
import torch

from flodl_b200 import nn, ops
from flodl_b200.autograd import Variable
from flodl_b200.tensor import TensorError


def normal(*shape, seed=0, **kw):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64, **kw)


def definition(q, k, v, allowed, add, scale):
    """One query at a time over the keys that take part."""
    B, Sq, H, D = q.shape
    group = H // k.shape[2]
    o = torch.zeros_like(q)
    for b in range(B):
        for h in range(H):
            at = allowed[b].nonzero()[:, 0]
            for i in range(Sq):
                if len(at):
                    s = k[b, at, h // group] @ q[b, i, h] * scale + add[b, at]
                    o[b, i, h] = torch.softmax(s, 0) @ v[b, at, h // group]
    return o


@pytest.mark.parametrize("H,Hk", [(2, 2), (6, 2), (3, 1)])
def test_the_plain_form_is_the_definition(H, Hk):
    q, k, v = normal(2, 3, H, 8), normal(2, 5, Hk, 8, seed=1), normal(2, 5, Hk, 8, seed=2)
    every, none = torch.ones(2, 5, dtype=torch.bool), torch.zeros(2, 5, dtype=torch.float64)
    scale = 1 / math.sqrt(8)
    assert torch.allclose(ops.cross_attention(q, k, v), definition(q, k, v, every, none, scale), rtol=1e-10, atol=1e-12)
    mask = torch.tensor([[True, False, True, True, False], [False] * 5])
    want = definition(q, k, v, mask, none, 0.3)
    assert torch.allclose(ops.cross_attention(q, k, v, mask, 0.3), want, rtol=1e-10, atol=1e-12)
    assert (want[1] == 0).all()
    add = torch.where(mask, normal(2, 5, seed=3), float("-inf"))
    for m in (add, add[:, None, None]):
        assert torch.allclose(ops.cross_attention(q, k, v, m), definition(q, k, v, mask, add.masked_fill(~mask, 0), scale), rtol=1e-10, atol=1e-12)
    # whatever an absent key holds
    k2, v2 = k.clone(), v.clone()
    k2[0, 1], v2[0, 4], k2[1], v2[1] = float("nan"), float("inf"), float("-inf"), float("nan")
    assert torch.equal(ops.cross_attention(q, k2, v2, mask, 0.3), ops.cross_attention(q, k, v, mask, 0.3))


def test_gradients_against_differences():
    q, k, v = (normal(2, n, h, 4, seed=n, requires_grad=True) for n, h in ((3, 4), (5, 2), (5, 2)))
    mask = torch.tensor([[True, False, True, True, True], [False] * 5])
    assert torch.autograd.gradcheck(lambda *t: ops.cross_attention(*t, mask), (q, k, v))
    add = normal(2, 5, seed=9, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *t: ops.cross_attention(*t), (q, k, v, add))


def test_empty():
    q, k = torch.randn(2, 3, 2, 8, requires_grad=True), torch.randn(2, 0, 2, 8, requires_grad=True)
    o = ops.cross_attention(q, k, k)
    assert (o == 0).all()
    o.sum().backward()
    assert (q.grad == 0).all() and k.grad.shape == k.shape
    assert ops.cross_attention(q[:, :0], q, q).shape == (2, 0, 2, 8) and ops.cross_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 2, 8)


def test_refusals():
    q, k = torch.randn(2, 3, 4, 8), torch.randn(2, 5, 2, 8)
    bad = [
        lambda: ops.cross_attention(q[0], k, k), lambda: ops.cross_attention(q, k, k[:, :4]), lambda: ops.cross_attention(q, k[:1], k[:1]),
        lambda: ops.cross_attention(q, k[..., :4], k[..., :4]), lambda: ops.cross_attention(q[:, :, :3], k, k), lambda: ops.cross_attention(q, k.double(), k.double()),
        lambda: ops.cross_attention(q.long(), k.long(), k.long()), lambda: ops.cross_attention(q, k, k, torch.ones(2, 4).bool()),
        lambda: ops.cross_attention(q, k, k, torch.ones(3, 5).bool()), lambda: ops.cross_attention(q, k, k, torch.ones(2, 5).long()),
        lambda: ops.cross_attention(q, k, k, torch.ones(3, 5)), lambda: ops.cross_attention(q, k, k, torch.ones(2, 1, 3, 5)),
        lambda: ops.cross_attention(q, k, k, scale=float("nan")), lambda: ops.cross_attention(q[..., :0], k[..., :0], k[..., :0]),
        lambda: ops.cross_attention(q, k[:, :, :0], k[:, :, :0]),
    ]
    for call in bad:
        with pytest.raises(TensorError):
            call()
