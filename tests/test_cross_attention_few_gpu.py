"""Attention of a few queries over another sequence, a kernel of its own up to sixteen rows to a key head, on either side of that border; the checks and their bounds
are those of attention over another sequence."""
import pytest
import torch

from flodl_b200 import ops
from test_cross_attention_gpu import C, case, check  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sk", [1, 7, 15, 16, 17, 31, 32, 33, 63, 65, 129, 255, 257, 400])
def test_odd_lengths(C, Sk, D):
    check(C, *case(2, 1, Sk, 2, 2, D, seed=Sk))
    check(C, *case(1, 3, Sk, 4, 2, D, seed=Sk))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,H,Hk", [(1, 16, 1), (16, 2, 2), (15, 3, 3), (8, 4, 2), (9, 2, 2), (5, 6, 2), (1, 48, 1), (2, 24, 3), (17, 1, 1), (9, 4, 2), (20, 8, 8)])
def test_rows_to_a_key_head(C, Sq, H, Hk, D):
    q, k, v, do = case(2, Sq, 700, H, Hk, D, seed=Sq)
    check(C, q, k, v, do)
    mask = torch.arange(700, device="cuda")[None] < torch.tensor([[699], [1]], device="cuda")
    check(C, q, k, v, do, mask)


@pytest.mark.parametrize("Sq", [1, 20])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3, 2.0])
def test_scales(C, scale, Sq):
    q, k, v, do = case(2, Sq, 200, 4, 4, 64, seed=6, peak=0.5)
    check(C, q, k, v, do, None, scale)
    check(C, q, k, v, do, torch.arange(200, device="cuda")[None] % 3 > 0, scale)
    check(C, q, k, v, do, torch.where(torch.arange(200, device="cuda")[None] % 3 > 0, 0.25, float("-inf")), scale)


@pytest.mark.parametrize("value", [-1e4, -1e9, 3e4, torch.finfo(torch.float32).min, float("-inf")])
def test_rows_whose_keys_share_a_mask(C, value):
    q, k, v, do = case(2, 2, 300, 4, 2, 64, seed=5)
    add = torch.full((2, 300), value, device="cuda")
    add[1, :150] = 0.0
    check(C, q, k, v, do, add)


@pytest.mark.parametrize("D", [64, 128])
def test_masks_of_many_rows(C, D):
    """More tiles than CTAs; batches without a key; what absent keys hold reaches nothing, also with infinities in the queries of another batch."""
    q, k, v, do = case(160, 1, 90, 4, 4, D, seed=12)
    mask = torch.rand(160, 90, device="cuda", generator=torch.Generator(device="cuda").manual_seed(13)) < 0.5
    mask[::7] = False
    want = check(C, q, k, v, do, mask)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("-inf"), float("nan")
    for a, b in zip(want, check(C, q, k2, v2, do, mask)):
        assert torch.equal(a, b)
    q2 = q.clone()
    q2[0] = float("inf")                 # a batch without a key
    assert torch.equal(ops.cross_attention(q2, k2, v2, mask), want[0])


def test_nan_in_a_key_reaches_its_rows_only(C):
    q, k, v, _ = case(2, 1, 300, 8, 2, 64, seed=14)
    k[1, 123, 1] = float("nan")
    o = ops.cross_attention(q, k, v)
    assert o[1, :, 4:].isnan().all() and not o[0].isnan().any() and not o[1, :, :4].isnan().any()


MORE = [  # enough work for tiles of 128 rows
    (4, 120, 1300, 12, 12, 64), (2, 120, 1300, 8, 8, 128), (1, 200, 4100, 8, 8, 64),         # few of them over several blocks of keys: clusters, the last of eight
    (2, 100, 1400, 160, 80, 64), (1, 130, 20000, 2, 1, 128), (2, 400, 9000, 2, 1, 64),       # stretches
    (16, 129, 127, 24, 24, 64), (12, 300, 257, 16, 8, 128), (30, 33, 190, 24, 8, 64), (4, 640, 384, 8, 4, 64), (12, 70, 65, 48, 12, 128), (90, 17, 500, 16, 16, 64),
]


@pytest.mark.parametrize("shape", MORE, ids=str)
def test_tiles_of_128_rows(C, shape):
    B, Sq, Sk = shape[:3]
    q, k, v, do = case(*shape, seed=15)
    check(C, q, k, v, do)
    g = torch.Generator(device="cuda").manual_seed(16)
    mask = torch.rand(B, Sk, generator=g, device="cuda") < 0.6
    mask[0, Sk // 10:Sk // 2] = False
    if B > 1:
        mask[-1] = False
    want = check(C, q, k, v, do, mask)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    for a, b in zip(want, check(C, q, k2, v2, do, mask)):
        assert torch.equal(a, b)
    check(C, q, k, v, do, torch.where(mask, torch.randn(B, Sk, generator=g, device="cuda") - 1e4, float("-inf")))


@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
def test_scales_of_tiles_of_128_rows(C, scale):
    q, k, v, do = case(20, 50, 200, 24, 24, 64, seed=19, peak=0.5)
    check(C, q, k, v, do, None, scale)
    check(C, q, k, v, do, torch.arange(200, device="cuda")[None] < 170, scale)


@pytest.mark.parametrize("shape", [(1, 33, 64, 2, 2, 64), (2, 47, 130, 6, 2, 128), (1, 250, 90, 4, 4, 64), (3, 16, 40, 6, 1, 64), (1, 20, 9000, 1, 1, 64)], ids=str)
def test_several_tiles_of_rows(C, shape):
    B, Sq, Sk = shape[:3]
    q, k, v, do = case(*shape, seed=17)
    check(C, q, k, v, do)
    mask = torch.rand(B, Sk, device="cuda", generator=torch.Generator(device="cuda").manual_seed(18)) < 0.4
    mask[0, :Sk // 3] = False
    check(C, q, k, v, do, mask)
    check(C, q, k, v, do, torch.where(mask, torch.randn(B, Sk, device="cuda"), float("-inf")))


@pytest.mark.parametrize("shape", [(2, 1, 1500, 8, 8, 64), (1, 1, 9000, 2, 1, 128), (1, 2, 9000, 2, 2, 64), (160, 1, 90, 4, 4, 64)], ids=str)
def test_captured_tokens_replay_over_new_masks(C, shape):
    """Two graphs of one pool, in turn on two streams: a tile's parts meet in a cluster, by a second launch, or there is one."""
    B, Sq, Sk = shape[:3]
    q, k, v, _ = case(*shape, seed=21)
    masks = [torch.zeros(B, Sk, dtype=torch.bool, device="cuda"), torch.zeros(B, Sk, device="cuda")]
    side, pool, made = torch.cuda.Stream(), torch.cuda.graph_pool_handle(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m in masks:
            ops.cross_attention(q, k, v, m)
    torch.cuda.synchronize()
    for m in masks:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=side):
            o = ops.cross_attention(q, k, v, m)
        made.append((graph, o))
    g = torch.Generator(device="cuda").manual_seed(22)
    for i in range(6):
        masks[0].copy_(torch.rand(B, Sk, generator=g, device="cuda") < 0.2 * i)
        masks[1].copy_(torch.randn(B, Sk, generator=g, device="cuda").masked_fill_(~masks[0], float("-inf")))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        for (graph, o), m in zip(made, masks):
            with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
                graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, ops.cross_attention(q, k, v, m))
