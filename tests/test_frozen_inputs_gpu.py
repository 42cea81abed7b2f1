"""Gradients of some of the inputs: those that are asked for are right, whichever they are, and the others are not worked out."""
import itertools
import math

import pytest
import torch

from flodl_b200 import ops
from test_cross_attention_gpu import C, case, close, reference  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 5, 40, 2, 2, 64), (2, 1, 1500, 8, 8, 64), (3, 130, 300, 4, 2, 128), (2, 400, 9000, 2, 1, 64), (2, 100, 1400, 160, 80, 64), (70, 17, 200, 8, 8, 64)], ids=str)
def test_attention_over_another_sequence(C, shape):
    B, Sq, Sk = shape[:3]
    data = case(*shape, seed=1)
    mask = torch.rand(B, Sk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) < 0.6
    mask[0, Sk // 4:Sk // 2] = False
    mask[-1] = False
    for m in (None, mask):
        want = dict(zip("qkv", reference(*data, m, 1 / math.sqrt(shape[-1]))[1:]))
        for names in ("q", "k", "v", "qk", "qv", "kv"):
            ts = {n: t.detach().requires_grad_(n in names) for n, t in zip("qkv", data)}
            o = ops.cross_attention(*ts.values(), m)
            got = torch.autograd.grad(o, [ts[n] for n in names], data[3], retain_graph=True)
            for n, g, again in zip(names, got, torch.autograd.grad(o, [ts[n] for n in names], data[3])):
                close(g, *want[n], f"d{n} of {names}")
                assert torch.equal(g, again)
    assert C.read_status(0) == 0


def test_what_is_not_wanted_is_not_worked_out(C):
    """A frozen source: the rows' share of the work alone, on all of the GPU."""
    q, k, v, do = case(8, 1024, 4096, 8, 8, 64, seed=3)

    def timed(*wanted):
        leaves = [t.detach().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
        o = ops.cross_attention(*leaves)
        best = math.inf
        for _ in range(6):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(3):
                torch.autograd.grad(o, [t for t in leaves if t.requires_grad], do, retain_graph=True)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best
    both = timed(True, True, True)
    # rows are three of the seven products, keys four
    assert timed(True, False, False) < 0.75 * both and timed(False, True, True) < 0.85 * both


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_positions(packed, norm):
    g = torch.Generator(device="cuda").manual_seed(4)
    heads = ((3, 4),) if packed else ((4,), (2,))
    x, dy = ([torch.randn(2, 9, *h, 64, device="cuda", generator=g).bfloat16() for h in heads] for _ in range(2))
    w = [torch.randn(64, device="cuda", generator=g) + 1 for _ in range(2)] if norm else []
    f = ops.rotary_frequencies(64, device="cuda")

    def grads(which):
        t = [v.detach().requires_grad_(i in which) for i, v in enumerate(x + w)]
        xs = t[0] if packed else tuple(t[:2])
        y = ops.qk_norm_rotary(xs, *t[len(x):], f) if norm else ops.rotary(xs, f)
        return torch.autograd.grad(y, [t[i] for i in which], dy[0] if packed else dy)
    n = len(x) + len(w)
    every = grads(range(n))
    for count in range(1, n):
        for which in itertools.combinations(range(n), count):
            assert all(torch.equal(a, every[i]) for a, i in zip(grads(which), which))


def test_one_tensor_for_all_inputs():
    """Its gradient is the sum of three, one by one and in a batch, which goes by the plain form."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x, do = torch.randn(2, 9, 2, 64, device="cuda", generator=g).bfloat16(), torch.randn(3, 2, 9, 2, 64, device="cuda", generator=g).bfloat16()
    for leaf in (True, False):
        t = x.clone().requires_grad_()
        used = t if leaf else t * 1
        o = ops.cross_attention(used, used, used)
        one = [torch.autograd.grad(o, t, d, retain_graph=True)[0] for d in do]
        every = torch.autograd.grad(o, t, do, is_grads_batched=True)[0]
        for d, a, b in zip(do, one, every):
            want = torch.autograd.grad(ops.cross_attention(*[(w := x.double().requires_grad_())] * 3), w, d.double())[0]
            # three gradients of bf16 with P, dS and D rounded before them, or rounded only themselves
            assert (a.double() - want).norm() <= 6 * 2.0 ** -8 * want.norm() and (b.double() - want).norm() <= 3 * 2.0 ** -8 * want.norm()
