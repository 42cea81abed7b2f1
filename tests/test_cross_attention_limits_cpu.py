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


MASKS = [(torch.float64, -1e300), (torch.float64, torch.finfo(torch.float64).min), (torch.float64, 1e300), (torch.float32, torch.finfo(torch.float32).min),
         (torch.float32, torch.finfo(torch.float32).max), (torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.float16, torch.finfo(torch.float16).min),
         (torch.float64, -1e9), (torch.float32, -1e9), (torch.float32, 1e6)]


@pytest.mark.parametrize("kind,value", MASKS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_an_addend_that_a_row_shares(dtype, kind, value):
    """It costs the scores no bits, beyond 2^100 it takes their place, as in 64 bits; a finite one leaves no key absent, -inf does."""
    q, k, v = (normal(2, n, 2, 8, seed=n + i, dtype=dtype).requires_grad_() for i, n in enumerate((4, 40, 40)))
    add = torch.full((2, 40), value, dtype=kind)
    add[:, 30:] = float("-inf")
    add[1, :10] = 0.0
    got = ops.cross_attention(q, k, v, add)
    keep = torch.ones(2, 40, dtype=torch.bool)
    keep[:, 30:] = False
    # row 1: what is 60000 or more behind the others has a probability of zero
    keep[1, 10 if value < 0 else 0:30] = value > 0
    keep[1, :10] = value < 0
    wide = [t.detach().double().requires_grad_() for t in (q, k, v)]
    want = ops.cross_attention(*wide, keep)
    if abs(value) >= 2.0 ** 100:
        same = ops.cross_attention(wide[0] * 0, *wide[1:], keep)
        want = torch.cat((same[:1], want[1:] if value < 0 else same[1:]))
    # fp32 sums of 40 products of the order of ten, and the rounding of the result
    assert got.dtype == dtype and torch.allclose(got.double(), want, rtol=torch.finfo(dtype).eps, atol=2.0 ** -18)
    # a score that the addend has replaced still has its gradient: nothing says where a sum is rounded
    assert all(g.abs().max() > 0 and g.isfinite().all() for g in torch.autograd.grad(got.sum(), (q, k, v)))


def test_beyond_all_scores_the_largest_addend_decides():
    q, k, v = (normal(1, n, 1, 8, seed=n + i) for i, n in enumerate((2, 3, 3)))
    for add in ([-2e300, -1e300, -2e300], [1e31, 1.0000001e31, -1e31], [-1e38, 5.0, -1e300]):
        assert torch.equal(ops.cross_attention(q, k, v, torch.tensor([add], dtype=torch.float64))[0], v[0, 1].expand(2, 1, 8))


def test_small_differences_behind_a_large_addend_stay():
    """A 64-bit mask is not rounded to 32 bits before its rows' largest has left it."""
    q, k, v = (normal(2, n, 2, 8, seed=n + i) for i, n in enumerate((4, 40, 40)))
    fine = normal(2, 40, seed=5, dtype=torch.float64)
    # 2^30 away a 64-bit value is known to 2^-23
    assert torch.allclose(ops.cross_attention(q, k, v, fine - 2.0 ** 30), ops.cross_attention(q, k, v, fine), rtol=0, atol=2.0 ** -18)


def test_gradients_of_masks_with_shared_addends():
    q, k, v = (normal(1, n, 1, 4, seed=n + i, dtype=torch.float64) for i, n in enumerate((3, 5, 5)))
    add = torch.tensor([[100.0, 101.0, 99.5, float("-inf"), 100.25]], dtype=torch.float64)
    keep = add > float("-inf")
    assert torch.autograd.gradcheck(lambda m: ops.cross_attention(q, k, v, torch.where(keep, m, float("-inf"))), add.masked_fill(~keep, 0.0).requires_grad_())


def test_absent_keys_get_no_gradient_from_rows_that_are_no_numbers():
    q, k, v, do = (normal(2, n, 2, 8, seed=n + i) for i, n in enumerate((4, 6, 6, 4)))
    mask = torch.tensor([[True, False, True, True, False, True], [True, True, False, True, True, True]])
    q[0, 0, 0, 3], do[1, 2, 1, 5] = float("nan"), float("inf")
    for m in (mask, torch.zeros(2, 6).masked_fill(~mask, float("-inf"))):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        dk, dv = torch.autograd.grad(ops.cross_attention(*leaves, m), leaves[1:], do)
        assert (dk[~mask] == 0).all() and (dv[~mask] == 0).all() and dk[0, 0, 0].isnan().all()
