"""Attention over another sequence at the limits of what scores and masks may hold: the plain form."""
import pytest
import torch

from flodl_b200 import ops


def normal(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_scores_that_are_all_minus_infinity_are_not_rows_without_a_key(dtype):
    """Their softmax is NaN; a batch row without a key has zeros; one key with a score among them carries the row."""
    q, k, v = (normal(3, n, 2, 8, seed=n + i, dtype=dtype) for i, n in enumerate((4, 6, 6)))
    q, k[:, :, 0] = q.abs(), float("-inf")
    k[1, 2, 0] = 1.0
    mask = torch.ones(3, 6, dtype=torch.bool)
    mask[2] = False
    mask[0, 3:] = False
    for o in (ops.cross_attention(q, k, v, mask), ops.cross_attention(q, k, v, torch.zeros(3, 6).masked_fill(~mask, float("-inf")))):
        assert o[0, :, 0].isnan().all() and not o[0, :, 1].isnan().any() and (o[2] == 0).all()
        assert torch.equal(o[1, :, 0], v[1, 2, 0].expand(4, 8))
    assert ops.cross_attention(q, k, v)[[0, 2], :, 0].isnan().all()
