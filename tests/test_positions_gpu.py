"""Rotary positions and normalised queries and keys on the GPU against the definition in 64 bits.

Bounds. One rounding to the result's type is half a step, `finfo.eps / 2` of the value. Before it the kernel works in fp32 (u = 2^-24 a step's half): a turn takes sine and cosine
(2 u each, from an angle within u of half a turn, 3.2 u), two products and a sum, 8 u of the pair's size; the norm adds a sum of squares over at most 512 values in
shuffles and chains (16 u), a reciprocal root (2^-22 = 4 u) and two products: 24 u of n w. The gradient subtracts n mean(w g n) from w g: 64 u of the sizes of both."""
import pytest
import torch

from flodl_b200 import ops

pytestmark = pytest.mark.gpu

@pytest.fixture(autouse=True)
def kernels_only(monkeypatch):
    """No call of these tests is answered by the plain form unnoticed."""
    from flodl_b200.ops import position

    def refuse(*a):
        raise AssertionError("the plain form was taken")
    monkeypatch.setattr(position, "_turn", refuse)


U = 2.0 ** -24
EPS = 1e-6


def turned(x, angles, interleaved, back=False):
    p = angles.shape[-1]
    r, rest = x[..., :2 * p], x[..., 2 * p:]
    z = torch.complex(r[..., 0::2], r[..., 1::2]) if interleaved else torch.complex(r[..., :p], r[..., p:])
    z = z * torch.exp((-1j if back else 1j) * angles)
    y = torch.stack((z.real, z.imag), -1).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((y, rest), -1)


def close(got, want, size, steps):
    """`size`: of what the fp32 error is counted in, broadcast to the values."""
    bound = want.abs() * (torch.finfo(got.dtype).eps / 2) + steps * U * size + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = (got.double() - want).abs()
    assert got.shape == want.shape and (off <= bound).all(), f"{(off / bound).max().item():.3g} times the bound"


def angles(f, B, S, pos, offset=0):
    p = torch.arange(S, device="cuda")[None] if pos is None else pos
    return (p + offset).double()[..., None, None] * f


def check_rotary(x, dy, f, pos, offset, interleaved):
    """Forward and gradient of one call; x, dy: a tensor (4-D, or packed 5-D) or a pair."""
    pair = not torch.is_tensor(x)
    xs, dys = (x, dy) if pair else ((x,), (dy,))
    leaves = [t.detach().requires_grad_() for t in xs]
    y = ops.rotary(tuple(leaves) if pair else leaves[0], f, pos, offset, interleaved)
    with torch.no_grad():
        again = ops.rotary(x, f, pos, offset, interleaved)
    ys = y if pair else (y,)
    for a, b in zip(ys, again if pair else (again,)):
        assert torch.equal(a, b)
    gs = torch.autograd.grad(ys, leaves, dys)
    for t, d, y, g in zip(xs, dys, ys, gs):
        a = angles(f, *t.shape[:2], pos, offset)
        for seg in range(3 if t.dim() == 5 else 1):
            t1, d1, y1, g1 = ((v[:, :, seg] if t.dim() == 5 else v) for v in (t, d, y, g))
            if seg == 2:
                assert torch.equal(t1, y1) and torch.equal(d1, g1)
                continue
            for src, got, back in ((t1, y1, False), (d1, g1, True)):
                size = src.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
                close(got, turned(src.double(), a, interleaved, back), size, 8)


SHAPES = [  # B, S, H, Hk, D, rot, positions
    (1, 1, 1, 1, 64, 64, "own"), (16, 1, 8, 8, 64, 64, "own"), (2, 33, 12, 12, 64, 32, None), (3, 7, 8, 2, 128, 128, "row"), (2, 130, 5, 5, 80, 40, None),
    (1, 515, 3, 1, 96, 48, "own"), (2, 19, 2, 2, 256, 256, None), (2, 9, 4, 4, 64, 6, None), (1, 3, 2, 1, 10, 10, "own"), (700, 3, 1, 1, 64, 64, "row"),
]


def case(B, S, H, Hk, D, positions, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = [torch.randn(B, S, h, D, generator=g, device="cuda").to(dtype) for h in (H, Hk, H, Hk)]
    pos = None
    if positions:
        pos = torch.randint(-5, 200000, (B if positions == "own" else 1, 1), generator=g, device="cuda") + torch.arange(S, device="cuda")
        pos = pos if positions == "own" else pos[0]
    return made[:2], made[2:], pos


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary(shape, dtype, interleaved):
    B, S, H, Hk, D, rot, positions = shape
    x, dy, pos = case(B, S, H, Hk, D, positions, dtype)
    f = ops.rotary_frequencies(rot, device="cuda")
    check_rotary(tuple(x), tuple(dy), f, pos, 3, interleaved)
    check_rotary(x[0], dy[0], f, pos, 0, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 64), (20, 20)])
def test_rotary_layouts(D, rot, interleaved):
    """Packed projections, heads before positions, slices, rows off a 16-byte boundary, an inner stride, gradients of one value for all."""
    g = torch.Generator(device="cuda").manual_seed(D)
    f = ops.rotary_frequencies(rot, device="cuda")

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda").bfloat16()
    check_rotary(normal(2, 37, 3, 4, D), normal(2, 37, 3, 4, D), f, None, 5, interleaved)
    bhsd = normal(2, 4, 37, D).transpose(1, 2)
    check_rotary(bhsd, normal(37, 2, 4, D).transpose(0, 1), f, None, 0, interleaved)
    packed = normal(2, 37, 3, 4, D)
    check_rotary((packed[:, :, 0], packed[:, ::1, 1, :2]), (normal(2, 37, 4, D), normal(2, 37, 2, D)), f, None, 0, interleaved)
    check_rotary(normal(2, 37, 4, D + 3)[..., 3:], normal(2, 37, 4, D + 2)[..., 2:], f, None, 0, interleaved)
    check_rotary(normal(2, 37, 4, 2 * D)[..., ::2], normal(1, 1, 1, 1).expand(2, 37, 4, D), f, None, 0, interleaved)


def check_norm(x, dy, wq, wk, f, pos, offset, interleaved):
    pair = not torch.is_tensor(x)
    xs, dys = (x, dy) if pair else ((x,), (dy,))
    leaves = [t.detach().requires_grad_() for t in xs]
    ws = [None if w is None else w.detach().requires_grad_() for w in (wq, wk)]
    y = ops.qk_norm_rotary(tuple(leaves) if pair else leaves[0], *ws, f, pos, offset, interleaved, eps=EPS)
    with torch.no_grad():
        again = ops.qk_norm_rotary(x, *ws, f, pos, offset, interleaved, eps=EPS)
    ys = y if pair else (y,)
    for a, b in zip(ys, again if pair else (again,)):
        assert torch.equal(a, b)
    gs = torch.autograd.grad(ys, leaves + [w for w in ws if w is not None], dys)
    twice = torch.autograd.grad(ops.qk_norm_rotary(tuple(leaves) if pair else leaves[0], *ws, f, pos, offset, interleaved, eps=EPS),
                                leaves + [w for w in ws if w is not None], dys)
    assert all(torch.equal(a, b) for a, b in zip(gs, twice))
    dws = list(gs[len(leaves):])
    rows = []
    for t, d, y, g in zip(xs, dys, ys, gs):
        if t.dim() == 5:
            assert torch.equal(t[:, :, 2], y[:, :, 2]) and torch.equal(d[:, :, 2], g[:, :, 2])
            rows += [tuple(v[:, :, i] for v in (t, d, y, g)) for i in range(2)]
        else:
            rows.append((t, d, y, g))
    for (t, d, y, g), w in zip(rows, ws):
        B, S, _, D = t.shape
        a = angles(f, B, S, pos, offset) if f is not None else torch.zeros(1, S, 1, 0, device="cuda", dtype=torch.float64)
        t, d = t.double(), d.double()
        wd = torch.ones(D, device="cuda", dtype=torch.float64) if w is None else w.detach().double()
        r = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)
        n = t * r
        close(y, turned(n * wd, a, interleaved), (n * wd).abs().amax(-1, keepdim=True) * 2 ** 0.5, 24)
        e = turned(d, a, interleaved, back=True)
        c = (e * wd * n).mean(-1, keepdim=True)
        # A turn's error is 8 u of the pair, of which e may be the small difference a cos - b sin: sizes are counted in the pairs of d, at most sqrt 2
        # of the row's largest value, and not in e.
        pair = d.abs().amax(-1, keepdim=True) * 2 ** 0.5
        size = r * pair * wd.abs().max() * (1 + n.abs().amax(-1, keepdim=True) * n.abs().mean(-1, keepdim=True))
        close(g, r * (e * wd - n * c), size, 64)
        if w is not None:       # chains of at most 64 rows a thread, 14 levels of pairs, 32 u of each term
            close(dws.pop(0), (e * n).sum((0, 1, 2)), (pair * n.abs()).sum((0, 1, 2)), 128)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm(shape, dtype, interleaved):
    B, S, H, Hk, D, rot, positions = shape
    x, dy, pos = case(B, S, H, Hk, D, positions, dtype)
    f = ops.rotary_frequencies(rot, device="cuda")
    wq, wk = (torch.randn(D, device="cuda") + 1 for _ in range(2))
    check_norm(tuple(x), tuple(dy), wq, wk, f, pos, 3, interleaved)
    check_norm(x[0], dy[0], wq, None, None, None, 0, interleaved)


@pytest.mark.parametrize("D,rot", [(64, 64), (128, 64), (20, 20)])
def test_norm_layouts(D, rot):
    g = torch.Generator(device="cuda").manual_seed(D)
    f = ops.rotary_frequencies(rot, device="cuda")
    w = torch.randn(2, D, generator=g, device="cuda")

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda").bfloat16()
    check_norm(normal(2, 1037, 3, 4, D), normal(2, 1037, 3, 4, D), w[0], w[1], f, None, 5, False)
    check_norm(normal(2, 4, 37, D).transpose(1, 2), normal(37, 2, 4, D).transpose(0, 1), w[0], None, f, None, 0, True)
    check_norm(normal(2, 37, 4, D + 3)[..., 3:], normal(2, 37, 4, D + 2)[..., 2:], None, None, f, None, 0, False)
    check_norm(normal(2, 37, 4, 2 * D)[..., ::2], normal(1, 1, 1, 1).expand(2, 37, 4, D), w[1], None, f, None, 0, False)


def test_rows_of_zeros_of_infinities_and_of_small_values():
    x = torch.randn(1, 4, 2, 64, device="cuda")
    x[0, 0] = 0
    x[0, 1, 0, 3] = float("inf")
    x[0, 2] *= 1e-18
    x[0, 3, 1, 5] = float("nan")
    x.requires_grad_()
    y = ops.qk_norm_rotary(x, None, None, ops.rotary_frequencies(64, device="cuda"))
    y.backward(torch.ones_like(y))
    assert (y[0, 0] == 0).all() and torch.isfinite(x.grad[0, 0]).all() and torch.isfinite(y[0, 2]).all()
    assert y[0, 1, 0].isnan().any() and torch.isfinite(y[0, 1, 1]).all()            # one row's trouble is its own
    assert y[0, 3, 1].isnan().any() and torch.isfinite(y[0, 3, 0]).all()


def test_replayed_with_other_positions():
    """A captured token step reads its positions anew."""
    q, k = torch.randn(3, 1, 4, 64, device="cuda").bfloat16(), torch.randn(3, 1, 2, 64, device="cuda").bfloat16()
    f, pos = ops.rotary_frequencies(64, device="cuda"), torch.zeros(3, 1, dtype=torch.int64, device="cuda")
    w = torch.ones(64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        ops.qk_norm_rotary(ops.rotary((q, k), f, pos), w, w, f, pos)
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad(), torch.cuda.graph(graph):
        y = ops.qk_norm_rotary(ops.rotary((q, k), f, pos), w, w, f, pos)
    for at in (5, 70000):
        pos.fill_(at)
        graph.replay()
        with torch.no_grad():
            want = ops.qk_norm_rotary(ops.rotary((q, k), f, pos), w, w, f, pos)
        assert all(torch.equal(a, b) for a, b in zip(y, want))


def test_many_tokens_of_many_heads():
    """Blocks of the norm's backward pass that walk over several tiles; 32-bit element offsets are passed."""
    x = torch.randn(1, 1, 64, 128, device="cuda").bfloat16().expand(3, 90000, 64, 128)
    f = ops.rotary_frequencies(128, device="cuda")
    dy = torch.randn(1, 1, 64, 128, device="cuda").bfloat16().expand(3, 90000, 64, 128)
    w = torch.ones(128, device="cuda", requires_grad=True)
    y = ops.qk_norm_rotary(x, w, None, f, interleaved=True)
    (dw,) = torch.autograd.grad(y, w, dy)
    row = slice(89990, 90000)
    a = angles(f, 3, 90000, None)[:, row]
    n = x[:, row].double()
    n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + EPS)
    close(y[:, row], turned(n, a, True), n.abs().amax(-1, keepdim=True) * 2 ** 0.5, 24)
    # dw: sum over positions of R^T dy n, in 64 bits, the rows of a position being the same in every batch
    total = torch.zeros(128, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    for s in range(0, 90000, 10000):
        d = dy[:1, s:s + 10000].double()
        e = turned(d, angles(f, 1, 90000, None)[:, s:s + 10000], True, back=True) * n[:1, :1]
        total += 3 * e.sum((0, 1, 2))
        size += 3 * (d.abs().amax(-1, keepdim=True) * 2 ** 0.5 * n[:1, :1].abs()).sum((0, 1, 2))
    # 270000 x 64 rows over 592 blocks of 16 rows at a time: chains of 1825 terms, each addition rounding its partial sum
    close(dw, total, size, 1825 + 64)


def test_refusals_of_devices():
    x = torch.randn(1, 2, 1, 8, device="cuda")
    with pytest.raises(RuntimeError):
        ops.rotary(x, ops.rotary_frequencies(8))
    with pytest.raises(RuntimeError):
        ops.rotary(x, ops.rotary_frequencies(8, device="cuda"), torch.arange(2))
    with pytest.raises(RuntimeError):
        ops.qk_norm_rotary(x, torch.ones(8))
