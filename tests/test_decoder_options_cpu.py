"""The decoder language model with rotary positions, normalised queries and keys and attention over a source: against the formulas written out in 64 bits,
gradients against differences, what positions and masks must and must not change, and the refusals."""
import pytest
import torch

from flodl_b200 import nn, ops
from flodl_b200.models.gpt import DecoderBlock, DecoderLM, DecoderLMConfig
from flodl_b200.autograd import Variable
from flodl_b200.tensor import TensorError

SMALL = dict(vocab_size=11, d_model=16, n_layers=2, n_heads=2, d_ff=12, max_seq=9)


def model(**kw):
    torch.manual_seed(3)
    m = DecoderLM(DecoderLMConfig(**{**SMALL, **kw}))
    for p in m.parameters():
        p.t.data = torch.randn_like(p.t, dtype=torch.float64) * 0.3 + (1.0 if p.t.dim() == 1 else 0.0)
    return m


def lin(m, x):
    return x @ m.weight.t.T + m.bias.t


def norm(m, x):
    return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * m.weight.t + m.bias.t


def gelu(x):
    return 0.5 * x * (1 + torch.erf(x / 2 ** 0.5))


def written_out(m, ids, source=None, keep=None):
    c = m.cfg
    B, S = ids.shape
    H, D = c.n_heads, c.d_model // c.n_heads
    x = m.tok.weight.t[ids]
    if not c.rotary_dim:
        x = x + m.pos.weight.t[:S]
    for b in m.blocks:
        h = norm(b.ln1, x)
        q, k, v = (lin(w, h).view(B, S, H, D) for w in (b.q, b.k, b.v))
        if c.qk_norm:
            q, k = (t / (t.pow(2).mean(-1, keepdim=True) + c.qk_norm_eps).sqrt() * w.weight.t for t, w in ((q, b.q_norm), (k, b.k_norm)))
        if c.rotary_dim:
            half = c.rotary_dim // 2
            a = torch.arange(S).double()[:, None, None] * c.rotary_base ** (-torch.arange(half).double() / half)
            e = torch.exp(1j * a)
            turned = []
            for t in (q, k):
                z = torch.complex(t[..., :half], t[..., half:2 * half]) * e
                turned.append(torch.cat((z.real, z.imag, t[..., 2 * half:]), -1))
            q, k = turned
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / D ** 0.5
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), float("-inf"))
        x = x + lin(b.o, torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(B, S, -1))
        if c.cross:
            q = lin(b.xq, norm(b.ln_x, x)).view(B, S, H, D)
            k, v = (lin(w, source).view(B, -1, H, D) for w in (b.xk, b.xv))
            s = torch.einsum("bqhd,bkhd->bhqk", q, k) / D ** 0.5
            if keep is not None:
                s = s.masked_fill(~keep[:, None, None], float("-inf"))
            x = x + lin(b.xo, torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(B, S, -1))
        x = x + lin(b.down, gelu(lin(b.up, norm(b.ln2, x))))
    return norm(m.ln_f, x) @ m.head.weight.t.T


@pytest.mark.parametrize("kw", [dict(), dict(rotary_dim=8), dict(rotary_dim=4, rotary_base=100.0), dict(qk_norm=True), dict(rotary_dim=8, qk_norm=True),
                                dict(cross=True), dict(rotary_dim=6, qk_norm=True, cross=True)], ids=str)
def test_logits_are_the_formulas(kw):
    m = model(**kw)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 11, (3, 7), generator=g)
    args = ()
    if kw.get("cross"):
        keep = torch.tensor([[True] * 5, [True, False, True, True, False], [False, True, False, False, False]])
        args = (torch.randn(3, 5, 16, generator=g, dtype=torch.float64), keep)
    got = m.forward(Variable.wrap(ids), *((Variable.wrap(args[0]), args[1]) if args else ())).t
    want = written_out(m, ids, *args)
    assert torch.allclose(got, want, rtol=1e-9, atol=1e-9)       # 64 bits; two layers of terms of the order of ten


def test_gradients_are_the_formulas():
    m = model(rotary_dim=8, qk_norm=True, cross=True)
    g = torch.Generator().manual_seed(6)
    ids, y = (torch.randint(0, 11, (2, 6), generator=g) for _ in range(2))
    source = torch.randn(2, 4, 16, generator=g, dtype=torch.float64, requires_grad=True)
    keep = torch.tensor([[True, True, False, True], [True, True, True, True]])
    ps = [p.t for p in m.parameters()]
    assert len(ps) == len({id(p) for p in ps}) == 3 + 1 + 2 * (4 + 8 + 4 + 2 + 2 + 8)
    got = torch.autograd.grad(m.loss(ids, y, source, keep).t, ps + [source])
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(written_out(m, ids, source, keep).flatten(0, 1), y.flatten()), ps + [source])
    for a, b in zip(got, want):
        # the loss may be taken in 32 bits: 2^-24 a rounding, some tens of them, relative to the largest
        assert torch.allclose(a, b, rtol=0, atol=1e-5 * max(b.abs().max().item(), 1e-3))
    assert not got[-1][0, 2].any() and got[-1][0, 1].any()


def test_rotary_model_has_no_longest_length_and_sees_only_distances():
    m = model(rotary_dim=8, n_layers=1)
    ids = torch.randint(0, 11, (1, 20), generator=torch.Generator().manual_seed(7))       # beyond max_seq
    assert m.forward(Variable.wrap(ids)).t.shape == (1, 20, 11)
    scaled = model(rotary_dim=8, n_layers=1, rotary_scaling="linear", rotary_factor=4.0)
    assert torch.equal(scaled.freqs, m.freqs / 4)
    assert all("pos" not in vars(x) for x in (m, scaled)) and m.freqs.dtype == torch.float64
    m.move_to_device("cpu")
    assert m.freqs.device.type == "cpu"


def test_defaults_are_the_model_as_it_was():
    a = DecoderLM(DecoderLMConfig(**SMALL))
    assert len(a.parameters()) == 2 + 2 + 1 + 2 * (4 + 8 + 4) and a.freqs is None
    assert [p.shape() for p in a.parameters()][:2] == [[11, 16], [9, 16]]


def test_refusals():
    ids = torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(TensorError, match="takes a source"):
        model(cross=True).hidden(ids)
    with pytest.raises(TensorError, match="takes a source"):
        model().hidden(ids, torch.zeros(2, 4, 16))
    for shape in ((1, 4, 16), (2, 4, 8), (2, 16)):
        with pytest.raises(TensorError, match="source must be"):
            model(cross=True).hidden(ids, torch.zeros(shape))
    with pytest.raises(TensorError, match="exceeds the heads"):
        model(rotary_dim=10)
    with pytest.raises(TensorError, match="even"):
        model(rotary_dim=7)
    with pytest.raises(TensorError, match="inside its model"):
        DecoderBlock(DecoderLMConfig(**SMALL, rotary_dim=8)).forward(Variable.wrap(torch.zeros(1, 2, 16)))
    with pytest.raises(TensorError, match="mask must be"):
        model(cross=True).hidden(ids, torch.zeros(2, 4, 16), torch.ones(2, 5, dtype=torch.bool))


@pytest.mark.parametrize("shape", [None, (1, 5), (3, 1, 1, 5), (1, 1, 1, 5), (4, 5), (3, 1, 4, 5), (3, 2, 4, 5)], ids=str)
def test_multihead_attention_over_another_length_is_what_it_was(shape):
    torch.manual_seed(0)
    mha = nn.MultiheadAttention(16, 2)
    q, s = torch.randn(3, 4, 16), torch.randn(3, 5, 16)
    mask = None if shape is None else (torch.arange(torch.Size(shape).numel()).reshape(shape) % 3 == 1).float()
    assert shape is None or mha._of_keys(mask, 3, 5) == (shape[-2] == 1 if len(shape) > 2 else shape[0] == 1)
    got = mha.forward_ext(*(Variable.wrap(t) for t in (q, s, s)), mask).t
    w = {n: (a.t, b.t) for n, (a, b) in mha.proj.items()}
    qh, kh, vh = ((t @ w[n][0].T + w[n][1]).unflatten(-1, (2, 8)).transpose(1, 2) for n, t in (("q_proj", q), ("k_proj", s), ("v_proj", s)))
    a = qh @ kh.transpose(-1, -2) * 8 ** -0.5
    if mask is not None:
        a = a.masked_fill(mask.bool(), float("-inf"))
    want = (a.softmax(-1) @ vh).transpose(1, 2).flatten(2) @ w["out_proj"][0].T + w["out_proj"][1]
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
