"""Positions for attention and attention over another sequence, as cases that can be timed and whose results can be compared.

Three operators of `flodl_b200.ops`: `rotary` (rotary positions on queries and keys), `qk_norm_rotary` (their RMS norm per head
with the rotation in the same pass) and `cross_attention` (queries over keys and values of another length, an encoder's states).
A case is a dict of plain values: `listed()` names the standing ones, `draw(rng)` gives more of the same ranges, `prepare` builds
what a program holds before the call, `run` is one pass (in plain torch, or through the framework where `own` is set), `exact` is
the same result from the definition in 64 bits, `work` is the least a pass has to read, write and multiply.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ the cases
def _rot(kind, batch, seq, heads, kv_heads, dim, rot, **kw):
    c = dict(kind=kind, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=False, packed=False,
             dtype="bf16", train=False, start=0, factor=1.0)
    c.update(kw)
    return c


def _cross(batch, q_len, k_len, heads, kv_heads, dim, padded=False, train=False, **kw):
    return dict(kind="cross", batch=batch, q_len=q_len, k_len=k_len, heads=heads, kv_heads=kv_heads, dim=dim, padded=padded, train=train, **kw)


def listed():
    return [
        # generation: the next token of 16 sequences, each at a position of its own; the launch is all there is
        _rot("rotary", 16, 1, 8, 8, 64, 64, start=1000, name="rotary_token"),
        # training: the packed projection of the decoder language model at its benchmark's batch
        _rot("rotary", 32, 256, 8, 8, 64, 64, packed=True, train=True, name="rotary_train"),
        # a long context far from its start: neighbours as pairs, half of each head, frequencies stretched by four, 32-bit activations
        _rot("rotary", 2, 8191, 12, 12, 64, 32, interleaved=True, dtype="fp32", start=120000, factor=4.0, name="rotary_far"),
        # generation with normalised queries and keys, four query heads to a key head
        _rot("qk_norm", 64, 1, 32, 8, 128, 128, start=5000, name="qk_norm_token"),
        # training: the packed projection of the decoder language model on its longer context
        _rot("qk_norm", 4, 1024, 8, 8, 64, 64, packed=True, train=True, name="qk_norm_train"),
        # training on long sequences with shared key heads
        _rot("qk_norm", 2, 4096, 32, 8, 128, 128, train=True, name="qk_norm_long"),
        # generation: one token of each of 16 sequences looks at its padded source
        _cross(16, 1, 1500, 8, 8, 64, padded=True, name="cross_token"),
        # generation over a very long source, keys and values shared by eight query heads
        _cross(4, 1, 32768, 32, 4, 128, name="cross_token_long"),
        # a short question over a document, odd sizes
        _cross(3, 77, 1031, 12, 12, 64, name="cross_question"),
        # training: the decoder language model's batch over padded sources of up to 509 tokens
        _cross(32, 256, 509, 8, 8, 64, padded=True, train=True, name="cross_train"),
        # scoring: texts over long sources, forward only
        _cross(8, 1024, 4096, 12, 12, 64, name="cross_score"),
        # training over long sources, four query heads to a key head
        _cross(2, 2048, 8192, 16, 4, 128, train=True, name="cross_train_long"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    kind = rng.choice(["rotary", "qk_norm", "cross", "cross"])
    train = rng.random() < 0.5
    if kind == "cross":
        q_len = 1 if not train and rng.random() < 0.4 else _log(rng, 2, 4096)
        kv = rng.choice([1, 2, 4, 8, 12])
        return _cross(_log(rng, 1, 32), q_len, _log(rng, 16, 32768), kv * rng.choice([1, 1, 2, 4]), kv, rng.choice([64, 128]),
                      padded=rng.random() < 0.5, train=train)
    seq = 1 if not train and rng.random() < 0.4 else _log(rng, 2, 8192)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    rot = rng.choice([dim, dim, dim // 2])
    packed = rng.random() < 0.4
    kv = rng.choice([1, 2, 4, 8, 12])
    return _rot(kind, _log(rng, 1, 64), seq, kv if packed else kv * rng.choice([1, 2, 4]), kv, dim, rot, interleaved=rng.random() < 0.4, packed=packed,
                dtype=rng.choice(["bf16", "bf16", "fp32"]), train=train, start=rng.choice([0, 1000, 120000]), factor=rng.choice([1.0, 4.0]))


def draw(rng):
    """One more case of the listed ones' ranges, no dearer than the dearest listed case of its kind."""
    while True:
        c = _one(rng)
        mine = work(c)
        top = [work(x) for x in listed() if x["kind"] == c["kind"]]
        if mine["flops"] <= max(t["flops"] for t in top) and mine["bytes"] <= max(t["bytes"] for t in top):
            return c


# ----------------------------------------------------------------------------------------------- the inputs
def _freqs(c):
    """base^(-2i / rot) over the stretch factor, radians per position."""
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64)
    return ((10000.0 ** (-i / c["rot"])) / c["factor"]).to(DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, dtype, grad=False):
        t = torch.randn(*shape, generator=g, device=DEV).to(dtype)
        return t.requires_grad_() if grad else t

    s = {"case": c}
    if c["kind"] == "cross":
        B, bf, train = c["batch"], torch.bfloat16, c["train"]
        s["q"] = normal(B, c["q_len"], c["heads"], c["dim"], dtype=bf, grad=train)
        s["k"] = normal(B, c["k_len"], c["kv_heads"], c["dim"], dtype=bf, grad=train)
        s["v"] = normal(B, c["k_len"], c["kv_heads"], c["dim"], dtype=bf, grad=train)
        s["mask"] = None
        if c["padded"]:      # True for the keys that take part: half of the longest source to all of it
            lengths = torch.randint((c["k_len"] + 1) // 2, c["k_len"] + 1, (B, 1), generator=g, device=DEV)
            s["mask"] = torch.arange(c["k_len"], device=DEV)[None, :] < lengths
        if train:
            s["dy"] = normal(B, c["q_len"], c["heads"], c["dim"], dtype=bf)
        return s
    B, S, D, dt, train = c["batch"], c["seq"], c["dim"], TYPES[c["dtype"]], c["train"]
    if c["packed"]:
        s["x"] = normal(B, S, 3, c["heads"], D, dtype=dt, grad=train)
        s["dy"] = normal(B, S, 3, c["heads"], D, dtype=dt) if train else None
    else:
        s["x"] = (normal(B, S, c["heads"], D, dtype=dt, grad=train), normal(B, S, c["kv_heads"], D, dtype=dt, grad=train))
        s["dy"] = (normal(B, S, c["heads"], D, dtype=dt), normal(B, S, c["kv_heads"], D, dtype=dt)) if train else None
    # positions of one sequence after another where there are starts to differ by, 0, 1, 2, ... otherwise
    s["positions"] = None
    if c["start"]:
        s["positions"] = torch.randint(0, c["start"], (B, 1), generator=g, device=DEV) + torch.arange(S, device=DEV)[None, :]
    s["freqs"] = _freqs(c)
    if c["kind"] == "qk_norm":
        s["wq"], s["wk"] = ((1 + 0.1 * torch.randn(D, generator=g, device=DEV)).requires_grad_(train) for _ in range(2))
    return s


# ------------------------------------------------------------------------------------------- the plain forms
def _angles(s):
    """cos and sin for each position and pair, [B or 1, S, 1, pairs]: angles in 64 bits, far positions times fast frequencies."""
    c, pos = s["case"], s["positions"]
    if pos is None:
        pos = torch.arange(c["seq"], device=DEV)[None, :]
    a = pos.double()[:, :, None, None] * s["freqs"]
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, rot, interleaved):
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return y if rest.shape[-1] == 0 else torch.cat((y, rest), dim=-1)


def _two(x):
    return (x[:, :, 0], x[:, :, 1]) if torch.is_tensor(x) else x


def _like(x, q, k):
    """Queries and keys back in the layout that they came in; the values of a packed tensor as they were."""
    if torch.is_tensor(x):
        return torch.stack((q.to(x.dtype), k.to(x.dtype), x[:, :, 2]), dim=2)
    return q.to(x[0].dtype), k.to(x[1].dtype)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    q, k = (t.detach().float() for t in _two(s["x"]))
    y = _like(s["x"], *(_rotate(t, cos, sin, c["rot"], c["interleaved"]) for t in (q, k)))
    if not c["train"]:
        return {"y": y}
    dq, dk = (t.float() for t in _two(s["dy"]))
    return {"y": y, "dx": _like(s["dy"], *(_rotate(t, cos, -sin, c["rot"], c["interleaved"]) for t in (dq, dk)))}


def _plain_norm(s):
    c = s["case"]
    cos, sin = _angles(s)
    out, dx, dw = [], [], []
    for i, (x, w) in enumerate(zip(_two(s["x"]), (s["wq"], s["wk"]))):
        x, w = x.detach().float(), w.detach()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        out.append(_rotate(n * w, cos, sin, c["rot"], c["interleaved"]))
        if c["train"]:
            g = _rotate(_two(s["dy"])[i].float(), cos, -sin, c["rot"], c["interleaved"])
            dw.append((g * n).sum((0, 1, 2)))
            g = g * w
            dx.append(r * (g - n * (g * n).mean(-1, keepdim=True)))
    y = _like(s["x"], *out)
    return {"y": y, "dx": _like(s["dy"], *dx), "dwq": dw[0], "dwk": dw[1]} if c["train"] else {"y": y}


def _plain_cross(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    B, Sq, Sk, D = c["batch"], c["q_len"], c["k_len"], c["dim"]
    scale = 1.0 / math.sqrt(D)
    q = s["q"].detach().float().transpose(1, 2).reshape(B, c["kv_heads"], group * Sq, D)       # a key head's queries together
    k, v = (s[n].detach().float().transpose(1, 2) for n in ("k", "v"))
    p = (q @ k.transpose(-1, -2)) * scale
    if s["mask"] is not None:
        p.masked_fill_(~s["mask"][:, None, None, :], float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p @ v

    def rows(t, heads):
        return t.reshape(B, heads, -1, D).transpose(1, 2).to(torch.bfloat16).contiguous()

    if not c["train"]:
        return {"o": rows(o, c["heads"])}
    do = s["dy"].float().transpose(1, 2).reshape(B, c["kv_heads"], group * Sq, D)
    ds = do @ v.transpose(-1, -2)
    ds = p * (ds - (do * o).sum(-1, keepdim=True)) * scale
    return {"o": rows(o, c["heads"]), "dq": rows(ds @ k, c["heads"]), "dk": rows(ds.transpose(-1, -2) @ q, c["kv_heads"]),
            "dv": rows(p.transpose(-1, -2) @ do, c["kv_heads"])}


# -------------------------------------------------------------------------------------- the framework's calls
def _own_rotary(s):
    from flodl_b200 import ops
    c = s["case"]
    y = ops.rotary(s["x"], s["freqs"], s["positions"], interleaved=c["interleaved"])
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dx": _grads(y, s["x"], s["dy"])}


def _own_norm(s):
    from flodl_b200 import ops
    c = s["case"]
    y = ops.qk_norm_rotary(s["x"], s["wq"], s["wk"], s["freqs"], s["positions"], interleaved=c["interleaved"], eps=EPS)
    if not c["train"]:
        return {"y": y}
    *dx, dwq, dwk = torch.autograd.grad(y, (*_as_tuple(s["x"]), s["wq"], s["wk"]), s["dy"])
    return {"y": y, "dx": dx[0] if torch.is_tensor(s["x"]) else tuple(dx), "dwq": dwq, "dwk": dwk}


def _own_cross(s):
    from flodl_b200 import ops
    o = ops.cross_attention(s["q"], s["k"], s["v"], s["mask"])
    if not s["case"]["train"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["dy"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _as_tuple(x):
    return (x,) if torch.is_tensor(x) else x


def _grads(y, x, dy):
    g = torch.autograd.grad(y, _as_tuple(x), dy)
    return g[0] if torch.is_tensor(x) else g


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "qk_norm": _own_norm, "cross": _own_cross}[kind](state)
    return {"rotary": _plain_rotary, "qk_norm": _plain_norm, "cross": _plain_cross}[kind](state)


# ------------------------------------------------------------------------------------------ the least of work
def work(case):
    c = case
    if c["kind"] == "cross":
        part = 0.75 if c["padded"] else 1.0              # the mean share of the keys that take part
        rows, keys = c["batch"] * c["heads"] * c["q_len"], c["batch"] * c["kv_heads"] * c["k_len"] * part
        product = 2.0 * c["batch"] * c["heads"] * c["q_len"] * c["k_len"] * part * c["dim"]
        if c["train"]:                                   # q, k, v and dO in; o, dq, dk, dv out; two products forward, five backward
            return {"bytes": 2.0 * c["dim"] * (4 * rows + 4 * keys), "flops": 7 * product}
        return {"bytes": 2.0 * c["dim"] * (2 * rows + 2 * keys), "flops": 2 * product}
    heads = 3 * c["heads"] if c["packed"] else c["heads"] + c["kv_heads"]
    n = float(c["batch"] * c["seq"] * heads * c["dim"])
    size = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "rotary":                            # x in, y out; dy in, dx out
        return {"bytes": n * size * (4 if c["train"] else 2), "flops": n * (6 if c["train"] else 3)}
    return {"bytes": n * size * (4 if c["train"] else 2), "flops": n * (20 if c["train"] else 7)}


# --------------------------------------------------------------------------------- the definition in 64 bits
def _turned(x, pos, freqs, rot, interleaved):
    """Each pair as a complex number, times e^(i angle)."""
    t = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos[..., None, None] * freqs)
    z = x[..., :rot]
    z = z.unflatten(-1, (rot // 2, 2)) if interleaved else z.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * t)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., rot:]), dim=-1)


def _exact_positions(s):
    c = s["case"]
    pos = (torch.arange(c["seq"], device=DEV)[None] if s["positions"] is None else s["positions"]).double()
    given = [t.detach().double().requires_grad_(c["train"]) for t in _two(s["x"])]
    w = [s[n].detach().double().requires_grad_(c["train"]) for n in ("wq", "wk")] if c["kind"] == "qk_norm" else []
    out = []
    for i, x in enumerate(given):
        if w:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w[i]
        out.append(_turned(x, pos, s["freqs"], c["rot"], c["interleaved"]))

    def back(like, a, b):
        return torch.stack((a, b, like[:, :, 2].double()), dim=2) if torch.is_tensor(like) else (a, b)

    y = back(s["x"], *(t.detach() for t in out))
    if not c["train"]:
        return {"y": y}
    g = torch.autograd.grad(out, given + w, [t.double() for t in _two(s["dy"])])
    r = {"y": y, "dx": back(s["dy"], g[0], g[1])}
    return {**r, "dwq": g[2], "dwk": g[3]} if w else r


def _exact_cross(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = {n: torch.empty_like(s[m], dtype=torch.float64) for n, m in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")) if n == "o" or c["train"]}
    for b in range(c["batch"]):
        for h in range(c["kv_heads"]):
            at = slice(h * group, (h + 1) * group)
            q = s["q"].detach()[b, :, at].double().requires_grad_(c["train"])
            k, v = (s[n].detach()[b, :, h].double().requires_grad_(c["train"]) for n in ("k", "v"))
            x = torch.einsum("qgd,kd->gqk", q, k) / math.sqrt(c["dim"])
            if s["mask"] is not None:
                x = x.masked_fill(~s["mask"][b], float("-inf"))
            o = torch.einsum("gqk,kd->qgd", torch.softmax(x, dim=-1), v)
            out["o"][b, :, at] = o.detach()
            if c["train"]:
                out["dq"][b, :, at], out["dk"][b, :, h], out["dv"][b, :, h] = torch.autograd.grad(o, (q, k, v), s["dy"][b, :, at].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_cross(s) if case["kind"] == "cross" else _exact_positions(s)
