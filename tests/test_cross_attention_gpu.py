"""Attention over another sequence on the GPU against the definition in 64 bits.

Bounds, with h = 2^-8 the most that one rounding to bf16 moves a value and t = 2^-12 what the fp32 scores, exponentials and sums of up to some thousand terms may add to a
probability. P is rounded once and so is the result:           |o|  <= (h + t) sum p |v| + h |o|,   |dv| <= (h + t) sum p |dO| + h |dv|.
D = rowsum(dO o) comes from the rounded o:                     eD   =  sum |dO| ((h + t) sum p |v| + h |o|), and dP = dO v in fp32 within t sum |dO| |v|;
dS = P (dP - D) is rounded once:                               eS   =  (h + t) |dS| + p (eD + t sum |dO| |v|),   |dq| <= scale sum eS |k| + h |dq|,   |dk| <= scale sum eS |q| + h |dk|."""
import math

import pytest
import torch

from flodl_b200 import ops

pytestmark = pytest.mark.gpu

H_, T_ = 2.0 ** -8, 2.0 ** -12


@pytest.fixture(scope="module")
def C():
    from flodl_b200 import _ext
    return _ext.require()


def close(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound + 1e-30)
    assert got.shape == want.shape and not bad.any(), f"{what}: {(off / (bound + 1e-30)).nan_to_num(1e9).max().item():.3g} times the bound, {int(bad.sum())} values"


def reference(q, k, v, do, mask, scale):
    """(o, dq, dk, dv) and how far each may be off, in 64 bits. Keys at False or -inf are taken out before anything is multiplied."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    g = H // Hk
    absent = torch.zeros(B, Sk, dtype=torch.bool, device=q.device)
    add = torch.zeros(B, Sk, dtype=torch.float64, device=q.device)
    if mask is not None:
        m = mask.reshape(mask.shape[0], Sk).expand(B, Sk)
        absent = ~m if m.dtype == torch.bool else m == float("-inf")
        if m.dtype != torch.bool:
            add = m.double().masked_fill(absent, 0.0)
    q5, do5 = (t.double().reshape(B, Sq, Hk, g, D).permute(0, 2, 3, 1, 4) for t in (q, do))              # [B, Hk, g, Sq, D]
    k4, v4 = (t.double().permute(0, 2, 1, 3).masked_fill(absent[:, None, :, None], 0.0)[:, :, None] for t in (k, v))       # [B, Hk, 1, Sk, D]
    s = (q5 @ k4.transpose(-1, -2)) * scale + add[:, None, None, None]
    s = s.masked_fill(absent[:, None, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = p @ v4
    eo = (H_ + T_) * (p @ v4.abs()) + H_ * o.abs()
    dp = do5 @ v4.transpose(-1, -2)
    ds = p * (dp - (do5 * o).sum(-1, keepdim=True))
    es = (H_ + T_) * ds.abs() + p * ((do5.abs() * eo).sum(-1, keepdim=True) + T_ * (do5.abs() @ v4.abs().transpose(-1, -2)))
    a = abs(scale)
    dq, edq = scale * (ds @ k4), a * (es @ k4.abs())
    dk, edk = scale * (ds.transpose(-1, -2) @ q5).sum(2), a * (es.transpose(-1, -2) @ q5.abs()).sum(2)
    dv, edv = (p.transpose(-1, -2) @ do5).sum(2), (H_ + T_) * (p.transpose(-1, -2) @ do5.abs()).sum(2)

    def rows(t):
        return t.permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D)

    def cols(t):
        return t.permute(0, 2, 1, 3)
    return ((rows(o), rows(eo)), (rows(dq), rows(edq + H_ * dq.abs())), (cols(dk), cols(edk + H_ * dk.abs())), (cols(dv), cols(edv + H_ * dv.abs())))


def check(C, q, k, v, do, mask=None, scale=None):
    C.clear_status(0)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.cross_attention(*leaves, mask, scale)
    ops.FLAGS.count_launches, ops.FLAGS.launches = True, 0
    with torch.no_grad():
        assert torch.equal(o, ops.cross_attention(q, k, v, mask, scale))
    ops.FLAGS.count_launches = False
    assert ops.FLAGS.launches == 1                 # the kernel, not the plain form
    got = (o, *torch.autograd.grad(o, leaves, do, retain_graph=True))
    for a, b in zip(got[1:], torch.autograd.grad(o, leaves, do)):
        assert torch.equal(a, b)                   # sums in one order
    assert C.read_status(0) == 0
    want = reference(q, k, v, do, mask, 1 / math.sqrt(q.shape[-1]) if scale is None else scale)
    for name, x, (y, bound) in zip(("o", "dq", "dk", "dv"), got, want):
        close(x, y, bound, name)
    return got


def case(B, Sq, Sk, H, Hk, D, seed=0, peak=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes = ((B, Sq, H, D), (B, Sk, Hk, D), (B, Sk, Hk, D), (B, Sq, H, D))
    q, k, v, do = (torch.randn(*s, generator=g, device="cuda") for s in shapes)
    return [t.bfloat16() for t in (q * peak, k, v, do)]


SHAPES = [  # B, Sq, Sk, H, Hk, D
    (1, 1, 1, 1, 1, 64), (1, 1, 129, 2, 2, 64), (2, 3, 64, 4, 4, 128), (2, 128, 128, 2, 2, 64), (1, 129, 127, 3, 3, 64), (2, 77, 1031, 4, 4, 64),
    (1, 300, 257, 4, 2, 128), (2, 33, 190, 6, 2, 64), (1, 5, 700, 32, 1, 64), (1, 70, 65, 12, 3, 128), (3, 1, 500, 16, 4, 128), (1, 640, 384, 2, 1, 64),
    (1, 1, 1200, 2, 2, 128), (2, 150, 900, 2, 2, 128), (2, 9, 1300, 4, 4, 64),        # few tiles over several blocks of keys: clusters
    (1, 2, 4100, 8, 8, 64), (1, 2, 4100, 8, 8, 128),                                  # ... of eight
    (2, 1, 1400, 160, 80, 64),                                                       # more tiles than clusters for them: stretches
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_no_mask(C, shape):
    check(C, *case(*shape))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_bool_mask(C, shape):
    """Lengths, holes, a batch without any key; what the absent keys hold is infinities and NaN."""
    B, Sq, Sk = shape[:3]
    q, k, v, do = case(*shape, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    mask = torch.rand(B, Sk, generator=g, device="cuda") < 0.7
    mask[0] = torch.arange(Sk, device="cuda") < max(1, Sk * 2 // 3)
    if B > 1:
        mask[1] = False
    want = check(C, q, k, v, do, mask)
    if B > 1:
        assert (want[0][1] == 0).all() and (want[1][1] == 0).all() and (want[2][1] == 0).all() and (want[3][1] == 0).all()
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    for a, b in zip(want, check(C, q, k2, v2, do, mask[:, None, None])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_added_mask(C, shape):
    B, Sq, Sk = shape[:3]
    q, k, v, do = case(*shape, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    add = torch.randn(B, Sk, generator=g, device="cuda")
    add[:, ::5] = float("-inf")
    add[:, 1::7] = -1e4
    add[:, -1] = torch.finfo(torch.float32).min
    check(C, q, k, v, do, add)
    check(C, q, k, v, do, add[:1].half().clamp(-60000, 60000))


@pytest.mark.parametrize("value", [-1e4, -1e9, 3e4, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, float("-inf")])
def test_rows_whose_keys_share_a_mask(C, value):
    """The row's maximum leaves the mask before the scores lose their bits to it; beyond 2^100 the mask takes the score's place, as in 64 bits."""
    q, k, v, do = case(2, 40, 300, 4, 2, 64, seed=5)
    add = torch.full((2, 300), value, device="cuda")
    add[1, :150] = 0.0
    check(C, q, k, v, do, add)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3, 2.0])
def test_scales(C, scale):
    q, k, v, do = case(2, 50, 200, 4, 4, 64, seed=6, peak=0.5)
    check(C, q, k, v, do, None, scale)
    check(C, q, k, v, do, torch.arange(200, device="cuda")[None] < 170, scale)


@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_over_many_keys(C, D):
    """Keys in parts, joined; and rows in parts for few keys, in the backward pass."""
    check(C, *case(1, 2, 9000, 2, 1, D, seed=7))
    check(C, *case(1, 3000, 100, 2, 1, D, seed=8))
    mask = torch.zeros(1, 9000, dtype=torch.bool, device="cuda")
    mask[0, 5000:5003] = True          # most parts have no key
    check(C, *case(1, 2, 9000, 2, 1, D, seed=9), mask)


@pytest.mark.parametrize("D", [64, 128])
def test_one_key_carries_a_row(C, D):
    q, k, v, do = case(2, 130, 260, 2, 2, D, seed=10, peak=4.0)
    check(C, q, k, v, do)


def test_layouts(C):
    """Heads before positions, slices of a packed projection, rows off a 16-byte boundary, an inner stride, one key sequence for every batch, gradients of one value."""
    g = torch.Generator(device="cuda").manual_seed(11)

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda").bfloat16()
    B, Sq, Sk, H = 2, 45, 150, 4
    q, kv, do = normal(B, H, Sq, 64).transpose(1, 2), normal(B, Sk, 2, H, 64), normal(B, Sq, H, 64)
    check(C, q, kv[:, :, 0], kv[:, :, 1], do)
    check(C, normal(B, Sq, H, 67)[..., 3:], normal(B, Sk, H, 128)[..., ::2], normal(B, Sk, H, 68)[..., 4:], do)
    check(C, normal(B, Sq, H, 64), normal(1, Sk, H, 64).expand(B, Sk, H, 64), normal(B, Sk, 1, 64).expand(B, Sk, H, 64), normal(1, 1, 1, 1).expand(B, Sq, H, 64))
    mask = (torch.arange(2 * Sk, device="cuda")[None] < 200)[:, ::2]
    check(C, q, kv[:, :, 0], kv[:, :, 1], do, mask)
    # gradients of broadcast inputs are summed over what they were broadcast to
    k1 = normal(1, Sk, H, 64).requires_grad_()
    o = ops.cross_attention(q, k1.expand(B, Sk, H, 64), kv[:, :, 1])
    o.backward(do)
    want = reference(q, k1.detach().expand(B, Sk, H, 64), kv[:, :, 1], do, None, 0.125)[2]
    close(k1.grad, want[0].sum(0, keepdim=True), want[1].sum(0, keepdim=True) + H_ * want[0].abs().sum(0, keepdim=True), "dk")


def test_offsets_beyond_32_bits(C):
    q = torch.randn(3, 1, 64, 128, device="cuda").bfloat16()
    k, v = (torch.randn(3, 90000, 64, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    C.clear_status(0)
    o = ops.cross_attention(q, k, v)
    assert C.read_status(0) == 0
    want = reference(q[2:, :, 60:], k[2:, :, 60:], v[2:, :, 60:], q[2:, :, 60:], None, 1 / math.sqrt(128))[0]
    close(o[2:, :, 60:], *want, "o")


def test_what_the_kernel_does_not_take():
    """Other types and head dims go by the plain form, with the same result."""
    for D, dtype, bound in ((64, torch.float32, 1e-5), (80, torch.bfloat16, 2e-2), (64, torch.float16, 3e-3)):
        q, k, v, do = (t.to(dtype) for t in case(2, 9, 33, 4, 2, D))
        o = ops.cross_attention(q, k, v, torch.arange(33, device="cuda")[None] < 20)
        want = reference(q, k, v, do, torch.arange(33, device="cuda")[None] < 20, 1 / math.sqrt(D))[0][0]
        assert o.dtype == dtype and (o.double() - want).abs().max() <= bound * want.abs().max()
    q, k, v, _ = case(2, 9, 33, 4, 2, 64)
    try:
        ops.set_native(False)
        plain = ops.cross_attention(q, k, v)
    finally:
        ops.set_native(True)
    assert (plain - ops.cross_attention(q, k, v)).abs().max() <= 2e-2


def test_second_derivatives_are_refused():
    q, k, v, do = (t.requires_grad_() for t in case(1, 4, 9, 2, 2, 64))
    o = ops.cross_attention(q, k, v)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, q, do, create_graph=True)


def test_captured_and_replayed_on_two_streams(C):
    """A forward and backward pass in a graph, replayed with other inputs; two graphs of one pool do not share what they work in; eager calls on a side stream beside them."""
    C.clear_status(0)
    q, k, v, do = case(2, 20, 3000, 4, 2, 64, seed=12)
    q, k, v = (t.requires_grad_() for t in (q, k, v))

    def step():
        o = ops.cross_attention(q, k, v)
        return (o, *torch.autograd.grad(o, (q, k, v), do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for seed in (13, 14):
        for t, n in zip((q, k, v, do), case(2, 20, 3000, 4, 2, 64, seed=seed)):
            with torch.no_grad():
                t.copy_(n)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        for g in graphs:
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, eager))
    assert C.read_status(0) == 0


def test_queries_and_keys_in_turn_over_a_source(C):
    """A decoder block's path: a packed projection normalised and turned, attention within, a second look at a padded source, and the way back."""
    g = torch.Generator(device="cuda").manual_seed(15)
    B, S, Sk, H, D = 2, 60, 210, 4, 64
    qkv = torch.randn(B, S, 3, H, D, generator=g, device="cuda").bfloat16().requires_grad_()
    kv = torch.randn(B, Sk, 2, H, D, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(2, D, device="cuda", requires_grad=True)
    f = ops.rotary_frequencies(D, device="cuda")
    mask = torch.arange(Sk, device="cuda")[None] < torch.tensor([[210], [100]], device="cuda")
    do = torch.randn(B, S, H, D, generator=g, device="cuda").bfloat16()

    def path():
        x = ops.attention(ops.qk_norm_rotary(qkv, w[0], w[1], f), causal=True)
        x = ops.cross_attention(ops.rotary(x, f), kv[:, :, 0], kv[:, :, 1], mask)
        return (x, *torch.autograd.grad(x, (qkv, kv, w), do))
    got = path()
    try:
        ops.set_native(False)
        want = path()
    finally:
        ops.set_native(True)
    # both are bf16 chains of three products and roundings: a few roundings of the typical value apart
    for a, b in zip(got, want):
        assert (a.double() - b.double()).norm() <= 4 * H_ * b.double().norm()
    assert (got[2][1, 100:] == 0).all()


def test_calls_that_look_at_more_than_memory():
    """Tangents and vmap go by the plain form, which knows them; both sides round their results to bf16 once."""
    g = torch.Generator().manual_seed(9)
    q, k, v, dv = (torch.randn(2, s, 2, 64, generator=g).bfloat16().cuda() for s in (3, 40, 40, 40))
    want, turn = ops.cross_attention(q, k, v), ops.cross_attention(q, k, dv)
    o, do = torch.func.jvp(lambda t: ops.cross_attention(q, k, t), (v,), (dv,))
    # P <= 1 rounded once by the kernel, the results once by either side, of sums that are at most the largest |v|
    assert (o - want).abs().max() <= 3 * H_ * v.abs().max() and (do - turn).abs().max() <= 3 * H_ * dv.abs().max()
    both = torch.func.vmap(lambda t: ops.cross_attention(q, k, t))(torch.stack((v, dv)))
    assert (both[1] - turn).abs().max() <= 3 * H_ * dv.abs().max()


@pytest.mark.parametrize("low", [-1e300, torch.finfo(torch.float64).min])
def test_lowest_values_of_a_64_bit_mask_stay_finite(low):
    """A row of them is a row of equal scores, not one without keys."""
    g = torch.Generator().manual_seed(10)
    q, k, v = (torch.randn(1, s, 1, 64, generator=g).bfloat16().cuda() for s in (3, 40, 40))
    mask = torch.full((1, 40), low, dtype=torch.float64, device="cuda")
    mask[0, 30:] = float("-inf")
    got = ops.cross_attention(q, k, v, mask)
    want = v[0, :30, 0].double().mean(0)
    assert ((got[0, :, 0].double() - want).abs() <= (H_ + T_) * v.abs().max().item() + H_ * want.abs()).all()
