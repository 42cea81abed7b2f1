"""The decoder language model with rotary positions, normalised queries and keys and attention over a source, and attention layers over another length, on the
kernels: no further from 64 bits than the same roundings in separate operators leave them, and one step captured and replayed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def all_native():
    """These sizes are small enough that, outside a capture, projections and norms would be left to PyTorch."""
    from flodl_b200.ops import core
    n = core.eager_min_numel()
    core.set_eager_min_numel(0)
    yield
    core.set_eager_min_numel(n)


OPTIONS = dict(rotary_dim=64, qk_norm=True, cross=True)


def build(dtype=None, **kw):
    from flodl_b200.models.gpt import DecoderLM, DecoderLMConfig
    torch.manual_seed(11)
    m = DecoderLM(DecoderLMConfig(vocab_size=512, d_model=128, n_layers=2, n_heads=2, d_ff=256, max_seq=128, **{**OPTIONS, **kw}), "cuda")
    if dtype:
        for p in m.parameters():
            p.t.data = p.t.data.to(dtype)
    return m


def batch(B=4, S=128, Sk=77):
    g = torch.Generator().manual_seed(12)
    ids = torch.randint(0, 512, (B, S + 1), generator=g).cuda()
    source = torch.randn(B, Sk, 128, generator=g).bfloat16().float().cuda()
    keep = (torch.arange(Sk)[None] < torch.tensor([77, 1, 64, 50])[:, None]).cuda()
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous(), source, keep


def rms(t):
    return t.double().pow(2).mean().sqrt().item()


@pytest.mark.parametrize("kw", [dict(), dict(qk_norm=False), dict(cross=False), dict(rotary_dim=32, cross=False, qk_norm=False)], ids=str)
def test_gradients_are_as_near_as_separate_operators(kw):
    """Both sides round the same places to bf16 (the plain side more: the turned halves, the probabilities), so the kernels' error is at most twice the plain
    side's, which leaves room for errors that fall differently; h = 2^-8 covers tensors whose plain error happens to be small."""
    from flodl_b200 import nn, ops
    ids, y, source, keep = batch()
    cross = kw.get("cross", True)

    def grads(m, src, guard):
        src = src.clone().requires_grad_()
        args = (src, keep) if cross else ()
        ps = [p.t for p in m.parameters()] + ([src] if cross else [])
        if guard:
            with nn.AutocastGuard(torch.bfloat16):
                return torch.autograd.grad(m.loss(ids, y, *args).t, ps)
        return torch.autograd.grad(m.loss(ids, y, *args).t, ps)
    ops.set_native(False)
    try:
        exact = grads(build(torch.float64, **kw), source.double(), False)
        plain = grads(build(**kw), source, True)
    finally:
        ops.set_native(True)
    ops.FLAGS.count_launches, ops.FLAGS.launches = True, 0
    got = grads(build(**kw), source, True)
    ops.FLAGS.count_launches = False
    assert ops.FLAGS.launches > 20
    for i, (a, b, e) in enumerate(zip(got, plain, exact)):
        assert a.shape == e.shape and rms(a.double() - e) <= 2 * rms(b.double() - e) + 2.0 ** -8 * rms(e), (i, rms(a.double() - e), rms(b.double() - e), rms(e))


def test_captured_step_replays_what_the_eager_step_gave():
    from flodl_b200 import nn
    from flodl_b200.parallel.engine import TrainEngine
    ids, y, source, keep = batch()
    m = build()
    m.set_training(True)
    before = [p.t.detach().clone() for p in m.parameters()]
    with nn.AutocastGuard(torch.bfloat16):
        eng = TrainEngine(m, lambda ps: nn.AdamW(ps, 0.0, 0.0), max_grad_norm=1.0)
        first = eng.step(lambda: m.loss(ids, y, source, keep)).item()
        eng.capture(lambda *a: m.loss(*a), [ids, y, source, keep], warmup=2)
        again = [eng.replay([ids, y, source, keep]).item() for _ in range(3)]
        shorter = keep & (torch.arange(77, device="cuda") < 40)
        other = eng.replay([ids, y, source, shorter]).item()
        eager = m.loss(ids, y, source, shorter).t.item()
        eng.check()
    assert again == [first] * 3 and other == eager != first          # at a learning rate of 0 nothing moves, and the masks are read anew
    assert all(torch.equal(p.t, b) for p, b in zip(m.parameters(), before))


@pytest.mark.parametrize("shape", [None, (1, 200), (3, 1, 1, 200), (40, 200)], ids=str)
def test_multihead_attention_over_another_length(shape):
    from flodl_b200 import nn, ops
    from flodl_b200.autograd import Variable
    torch.manual_seed(1)
    mha = nn.MultiheadAttention(128, 2, "cuda")
    q, s = torch.randn(3, 40, 128, device="cuda").bfloat16(), torch.randn(3, 200, 128, device="cuda").bfloat16()
    mask = None if shape is None else (torch.rand(shape, device="cuda") < 0.3).float()

    def run():
        with nn.AutocastGuard(torch.bfloat16):
            return mha.forward_ext(*(Variable.wrap(t) for t in (q, s, s)), mask).t
    ops.FLAGS.count_launches, ops.FLAGS.launches = True, 0
    got = run()
    n = ops.FLAGS.launches
    ops.set_native(False)
    try:
        plain = run()
    finally:
        ops.set_native(True)
        ops.FLAGS.count_launches = False
    assert n == (4 if shape == (40, 200) else 5)                       # four projections, and attention where the mask is one of keys
    w = {k: (a.t.double(), b.t.double()) for k, (a, b) in mha.proj.items()}
    qh, kh, vh = ((t.double() @ w[k][0].T + w[k][1]).unflatten(-1, (2, 64)).transpose(1, 2) for k, t in (("q_proj", q), ("k_proj", s), ("v_proj", s)))
    a = qh @ kh.transpose(-1, -2) * 64 ** -0.5
    if mask is not None:
        a = a.masked_fill(mask.bool(), float("-inf"))
    want = (a.softmax(-1) @ vh).transpose(1, 2).flatten(2) @ w["out_proj"][0].T + w["out_proj"][1]
    assert rms(got.double() - want) <= 1.5 * rms(plain.double() - want) + 2.0 ** -9 * rms(want)
