"""Attention over another sequence at the limits of what scores, masks and gradients may hold, on every way that a tile's rows take: one CTA, a cluster, parts that a
second launch joins, in tiles of sixteen and of 128 rows."""
import pytest
import torch

from flodl_b200 import ops
from test_cross_attention_gpu import C, case  # noqa: F401

pytestmark = pytest.mark.gpu

WAYS = [  # B, Sq, Sk, H, Hk, D
    (2, 2, 40, 2, 2, 64), (2, 1, 1500, 8, 8, 64), (2, 1, 9000, 2, 1, 128), (160, 1, 90, 4, 4, 64),          # tiles of sixteen rows
    (24, 130, 300, 16, 16, 64), (2, 120, 1300, 12, 12, 64), (2, 130, 20000, 2, 1, 128), (2, 400, 9000, 2, 1, 64), (2, 100, 1400, 160, 80, 64),
]


@pytest.mark.parametrize("shape", WAYS, ids=str)
def test_scores_that_are_all_minus_infinity_are_not_rows_without_a_key(C, shape):
    """Their softmax and its gradients are NaN; a batch row without a key has zeros; one key with a score among them carries the row."""
    B, Sq, Sk, H, Hk, D = shape
    q, k, v, do = case(*shape, seed=1)
    q, group = q.abs(), H // Hk
    k[0, :, 0] = float("-inf")
    want = v[0, Sk // 2, 0]
    mask = torch.ones(B, Sk, dtype=torch.bool, device="cuda")
    mask[0, :Sk // 3] = False
    mask[-1] = False
    for m in (None, mask, torch.zeros(B, Sk, device="cuda").masked_fill(~mask, float("-inf"))):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        o = ops.cross_attention(*leaves, m)
        dq, dk, dv = torch.autograd.grad(o, leaves, do)
        assert o[0, :, :group].isnan().all() and not o[0, :, group:].isnan().any() and not o[1:].isnan().any()
        assert dq[0, :, :group].isnan().all() and not dq[0, :, group:].isnan().any() and not dq[1:].isnan().any()
        there = slice(Sk // 3, None) if m is not None else slice(None)
        assert dk[0, there, 0].isnan().all() and dv[0, there, 0].isnan().all() and not dk[0, :, 1:].isnan().any() and not dv[1:].isnan().any()
        if m is not None:
            assert (o[-1] == 0).all() and (dq[-1] == 0).all() and (dk[-1] == 0).all() and (dv[-1] == 0).all()
    k[0, Sk // 2, 0] = 1.0
    for m in (None, mask):
        assert torch.equal(ops.cross_attention(q, k, v, m)[0, :, :group], want.expand(Sq, group, D))
    assert C.read_status(0) == 0


@pytest.mark.parametrize("shape", WAYS, ids=str)
def test_absent_keys_get_no_gradient_from_rows_that_are_no_numbers(C, shape):
    """A NaN in a query, an infinity in a result's gradient: what such rows give a key that takes part is no number, but an absent key still gets zeros."""
    B, Sq, Sk, H, Hk, D = shape
    q, k, v, do = case(*shape, seed=2)
    mask = torch.rand(B, Sk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.5
    mask[:, 0] = True
    q[0, 0, 0, 3] = float("nan")
    do[1, Sq - 1, H - 1, 5] = float("inf")
    for m in (mask, torch.zeros(B, Sk, device="cuda").masked_fill(~mask, float("-inf"))):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        dk, dv = torch.autograd.grad(ops.cross_attention(*leaves, m), leaves[1:], do)
        assert (dk[~mask] == 0).all() and (dv[~mask] == 0).all()
        assert dk[0, 0, 0].isnan().all() and dv[0, 0, 0].isnan().all() and not dv[1, 0, Hk - 1].isfinite().all()
    assert C.read_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 80), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("kind,value", [(torch.float64, -1e300), (torch.float64, -1e9), (torch.float64, 2.0 ** 30), (torch.float32, -1e9), (torch.float16, -60000.0)], ids=str)
def test_addends_that_a_row_shares(C, dtype, D, kind, value):
    """By the kernel and by the plain form, which takes the other types and heads: as by the plain form in 64 bits; of a 64-bit mask also what is behind a large one."""
    q, k, v, _ = (t.to(dtype) for t in case(2, 5, 300, 4, 2, D, seed=4))
    add = torch.full((2, 300), value, dtype=kind, device="cuda")
    add[0, 250:] = float("-inf")
    if kind == torch.float64 and abs(value) < 1e10:
        add[1] += torch.randn(300, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(5))
    got = ops.cross_attention(q, k, v, add)
    with torch.no_grad():
        ops.set_native(False)
        try:
            want = ops.cross_attention(*(t.double() for t in (q, k, v)), add)
        finally:
            ops.set_native(True)
    # bf16: P rounded once by the kernel, and the result; otherwise the result and fp32 sums
    bound = (2.0 ** -8 + 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -16) * v.double().abs().max() + torch.finfo(dtype).eps / 2 * want.abs()
    assert ((got.double() - want).abs() <= bound).all()
    assert C.read_status(0) == 0


def test_beyond_all_scores_the_largest_addend_decides(C):
    q, k, v, _ = case(1, 2, 3, 1, 1, 64, seed=6)
    for add in ([-2e300, -1e300, -2e300], [1e31, 1.0000001e31, -1e31], [-1e38, 5.0, -1e300]):
        assert torch.equal(ops.cross_attention(q, k, v, torch.tensor([add], dtype=torch.float64, device="cuda"))[0], v[0, 1].expand(2, 1, 64))
