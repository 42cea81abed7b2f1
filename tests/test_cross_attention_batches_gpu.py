"""Attention over another sequence for more batch rows than are looked through one after another, whose places among the tiles are searched for where a mask leaves
each its own number of blocks; the checks and their bounds are those of attention over another sequence."""
import pytest
import torch

from test_cross_attention_gpu import C, case, check  # noqa: F401

pytestmark = pytest.mark.gpu


def masks(B, Sk):
    g = torch.Generator(device="cuda").manual_seed(B + Sk)
    upto = torch.arange(Sk, device="cuda")[None]
    some = upto < torch.randint(1, Sk + 1, (B, 1), generator=g, device="cuda")
    yield some
    holes = torch.rand(B, Sk, generator=g, device="cuda") < 0.4
    holes[:B // 3] = False
    holes[B // 2::3] = False
    holes[-2:] = False
    yield holes
    last = torch.zeros(B, Sk, dtype=torch.bool, device="cuda")
    last[-1, Sk // 2] = True
    yield last
    yield torch.zeros(B, Sk, dtype=torch.bool, device="cuda")
    yield torch.where(some, torch.randn(B, Sk, generator=g, device="cuda"), float("-inf"))


@pytest.mark.parametrize("shape", [(64, 40, 700, 8, 8, 64), (65, 40, 700, 8, 8, 64), (66, 130, 300, 4, 2, 128), (70, 40, 3000, 1, 1, 64), (300, 17, 600, 8, 8, 64), (1025, 20, 130, 8, 4, 64), (1500, 3, 30, 2, 2, 64),
                                   (2047, 17, 33, 6, 6, 64)], ids=str)
def test_masks_of_many_batch_rows(C, shape):
    q, k, v, do = case(*shape, seed=1)
    for mask in masks(shape[0], shape[2]):
        check(C, q, k, v, do, mask)
