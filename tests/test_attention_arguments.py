"""What is no argument at all, for the operators on positions and attention over another sequence: the framework's own error, on a GPU as on the CPU."""
import numpy as np
import pytest
import torch

from flodl_b200 import ops
from flodl_b200.tensor import TensorError

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_positions(device):
    x, f = torch.randn(2, 3, 2, 64, device=device), ops.rotary_frequencies(64, device=device)
    packed = torch.randn(2, 3, 3, 2, 64, device=device)
    bad = [
        lambda: ops.rotary(x, None), lambda: ops.rotary(x, [0.1] * 32), lambda: ops.rotary(x, np.ones(32)), lambda: ops.rotary(x, f, [0, 1, 2]), lambda: ops.rotary(x, f, 3),
        lambda: ops.rotary(None, f), lambda: ops.rotary(3, f), lambda: ops.rotary({"q": x}, f), lambda: ops.rotary([packed], f), lambda: ops.rotary((packed, packed), f),
        lambda: ops.rotary(x, f, offset=2 ** 70), lambda: ops.rotary(x, f, offset=None), lambda: ops.rotary(x, f, offset=float("inf")), lambda: ops.rotary(x, f, offset="1"),
        lambda: ops.rotary(x, f, amplitude=None), lambda: ops.rotary(x, f, amplitude=float("inf")), lambda: ops.rotary(x, f, amplitude=torch.ones(2)),
        lambda: ops.qk_norm_rotary(None), lambda: ops.qk_norm_rotary(x, [1.0] * 64), lambda: ops.qk_norm_rotary(x, eps=None), lambda: ops.qk_norm_rotary(x, eps=float("nan")),
        lambda: ops.qk_norm_rotary(x, eps=float("inf")), lambda: ops.qk_norm_rotary([packed]), lambda: ops.qk_norm_rotary(x, None, None, [1.0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(TensorError):
            call()
            pytest.fail(f"call {i} was taken")
    # numbers that are not Python's own
    want = ops.rotary(x, f, offset=5, amplitude=2.0)
    for offset, amplitude in ((np.int64(5), np.float32(2)), (5.0, 2), (torch.tensor(5), torch.tensor(2.0))):
        assert torch.allclose(ops.rotary(x, f, offset=offset, amplitude=amplitude), want, rtol=0, atol=2.0 ** -20)
    assert all(torch.equal(a, b) for a, b in zip(ops.rotary([x], f), ops.rotary((x,), f)))


@pytest.mark.parametrize("device", DEVICES)
def test_attention_over_another_sequence(device):
    q, k = torch.randn(2, 3, 2, 64, device=device).bfloat16(), torch.randn(2, 5, 2, 64, device=device).bfloat16()
    bad = [
        lambda: ops.cross_attention(None, k, k), lambda: ops.cross_attention(q, None, k), lambda: ops.cross_attention(q, k, [1]), lambda: ops.cross_attention(q, k, k, [1, 1, 0, 1, 1]),
        lambda: ops.cross_attention(q, k, k, 1), lambda: ops.cross_attention(q, k, k, scale="1"), lambda: ops.cross_attention(q, k, k, scale=float("inf")),
        lambda: ops.cross_attention(q, k, k, scale=torch.ones(3)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(TensorError):
            call()
            pytest.fail(f"call {i} was taken")
    want = ops.cross_attention(q, k, k, scale=0.5)
    for scale in (np.float64(0.5), torch.tensor(0.5)):
        assert torch.equal(ops.cross_attention(q, k, k, scale=scale), want)
