"""Attention over another sequence with more work than fits the GPU at once."""
import pytest
import torch

from flodl_b200 import ops
from test_cross_attention_gpu import C, case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_repeat_under_load(C, D):
    """Warps of a block drift apart by a turn where its products wait for the memory that many blocks share."""
    q, k, v, do = case(2, 100, 1400, 160, 80, D, seed=20)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = ops.cross_attention(*leaves)
    want = torch.autograd.grad(o, leaves, do, retain_graph=True)
    assert all(t.isfinite().all() for t in want)
    for _ in range(40):
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(o, leaves, do, retain_graph=True)))
