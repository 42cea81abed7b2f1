"""Decoder-only transformer LM (scaled-up ddp-bench/src/models/gpt_nano.rs: pre-LayerNorm blocks,
GELU feed-forward, learned position embedding, untied vocabulary head).

    x = tok_emb[ids] + pos_emb
    per block:  x = x + dropout(attn(LN1(x)));  x = x + dropout(ffn(LN2(x)))
    logits = head(LN_f(x))

Kernel mapping on CUDA/bf16: each "add + dropout -> LayerNorm" is one fused kernel that returns
both the new residual stream and its normalised value; QKV is one GEMM (weights back to back in the
flat buffer), attention is the causal flash kernel, the FFN is two GEMMs with GELU / GELU' in the
epilogues, and `loss()` fuses the vocabulary projection with the softmax cross-entropy.

What the reference's model does not have, off by default: rotary positions in place of the position embedding (`rotary_dim`), RMS
norms of each query and key head (`qk_norm`), both one pass over the packed projection, and in every block attention over the states of
another sequence, behind the block's own attention (`cross`):  x = x + dropout(cross_attn(LNx(x), source))."""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional

import torch

from .. import ops as _ops
from ..autograd import Variable
from ..hf.transformer_layer import fused_rows
from ..nn.layers import Embedding, LayerNorm, Linear, RMSNorm
from ..nn.module import Module, Parameter
from ..tensor import TensorError


@dataclass
class DecoderLMConfig:
    vocab_size: int = 32000
    d_model: int = 512
    n_layers: int = 6
    n_heads: int = 8
    d_ff: int = 2048
    max_seq: int = 256
    dropout: float = 0.0
    layer_norm_eps: float = 1e-5
    rotary_dim: int = 0                       # columns of a head that turn; 0: a learned position embedding instead
    rotary_base: float = 10000.0
    rotary_scaling: Optional[str] = None      # of `ops.rotary_frequencies`, as is the factor; its original length is max_seq
    rotary_factor: float = 1.0
    qk_norm: bool = False
    qk_norm_eps: float = 1e-6
    cross: bool = False


class DecoderBlock(Module):
    def __init__(self, cfg: DecoderLMConfig, device=None):
        d = cfg.d_model
        self.cfg = cfg
        self.ln1, self.ln2 = LayerNorm(d, cfg.layer_norm_eps, device), LayerNorm(d, cfg.layer_norm_eps, device)
        self.q, self.k, self.v, self.o = (Linear(d, d, True, device) for _ in range(4))
        self.up, self.down = Linear(d, cfg.d_ff, True, device), Linear(cfg.d_ff, d, True, device)
        self._fused = None
        self.q_norm = self.k_norm = self.ln_x = None
        if cfg.qk_norm:
            self.q_norm, self.k_norm = (RMSNorm(d // cfg.n_heads, cfg.qk_norm_eps, device) for _ in range(2))
        if cfg.cross:
            self.ln_x = LayerNorm(d, cfg.layer_norm_eps, device)
            self.xq, self.xk, self.xv, self.xo = (Linear(d, d, True, device) for _ in range(4))

    def name(self): return "decoder_block"
    def sub_modules(self):
        m = [self.ln1, self.q, self.k, self.v, self.o, self.ln2, self.up, self.down]
        if self.q_norm is not None:
            m += [self.q_norm, self.k_norm]
        return m if self.ln_x is None else m + [self.ln_x, self.xq, self.xk, self.xv, self.xo]
    def fuse_groups(self): return [[self.q.weight, self.k.weight, self.v.weight], [self.q.bias, self.k.bias, self.v.bias]]

    def _qkv(self, h: torch.Tensor) -> torch.Tensor:
        B, S, d = h.shape
        H, D = self.cfg.n_heads, d // self.cfg.n_heads
        ws = [m.weight.t for m in (self.q, self.k, self.v)]
        bs = [m.bias.t for m in (self.q, self.k, self.v)]
        if h.is_cuda and getattr(ws[0], "_fb_flat", None) is not None:
            if self._fused is None or self._fused[0].data_ptr() != ws[0].data_ptr():
                fw, fb = fused_rows(ws), fused_rows(bs)
                self._fused = (fw, fb) if fw is not None and fb is not None else (ws[0], None)
            if self._fused[1] is not None:
                return _ops.linear(h, self._fused[0], self._fused[1]).view(B, S, 3, H, D)
        return _ops.packed_linear(h, ws, bs).view(B, S, 3, H, D)

    def _cross(self, h: torch.Tensor, source: torch.Tensor, source_mask) -> torch.Tensor:
        heads = (self.cfg.n_heads, h.shape[-1] // self.cfg.n_heads)
        q, k, v = (_ops.linear(t, m.weight.t, m.bias.t).unflatten(-1, heads) for m, t in ((self.xq, h), (self.xk, source), (self.xv, source)))
        return _ops.linear(_ops.cross_attention(q, k, v, source_mask).flatten(2), self.xo.weight.t, self.xo.bias.t)

    def forward_pair(self, delta, stream, freqs=None, source=None, source_mask=None):
        """`delta` is the previous sub-layer output not yet added to the residual `stream` (or None)."""
        c = self.cfg
        p = c.dropout
        if delta is None:
            h1, x = _ops.layer_norm(stream, self.ln1.weight.t, self.ln1.bias.t, c.layer_norm_eps), stream
        else:
            h1, x = _ops.layer_norm(delta, self.ln1.weight.t, self.ln1.bias.t, c.layer_norm_eps, residual=stream, p_drop=p,
                                    training=self.training, return_pre=True)
        B, S, d = x.shape
        qkv = self._qkv(h1)
        if self.q_norm is not None:
            qkv = _ops.qk_norm_rotary(qkv, self.q_norm.weight.t, self.k_norm.weight.t, freqs, eps=c.qk_norm_eps)
        elif freqs is not None:
            qkv = _ops.rotary(qkv, freqs)
        ctx = _ops.attention(qkv, causal=True, p_drop=0.0, training=self.training)
        a = _ops.linear(ctx.reshape(B, S, d), self.o.weight.t, self.o.bias.t)
        if self.ln_x is not None:
            hx, x = _ops.layer_norm(a, self.ln_x.weight.t, self.ln_x.bias.t, c.layer_norm_eps, residual=x, p_drop=p, training=self.training,
                                    return_pre=True)
            a = self._cross(hx, source, source_mask)
        h2, x2 = _ops.layer_norm(a, self.ln2.weight.t, self.ln2.bias.t, c.layer_norm_eps, residual=x, p_drop=p, training=self.training,
                                 return_pre=True)
        f = _ops.feed_forward(h2, self.up.weight.t, self.up.bias.t, self.down.weight.t, self.down.bias.t, "gelu")
        return f, x2

    def forward(self, x: Variable) -> Variable:
        if self.cfg.cross or self.cfg.rotary_dim:
            raise TensorError("a block with rotary positions or attention over a source runs inside its model")
        f, s = self.forward_pair(None, x.t)
        return Variable.wrap(s + _ops.dropout(f, self.cfg.dropout, self.training))


class DecoderLM(Module):
    def __init__(self, cfg: DecoderLMConfig, device=None):
        self.cfg = cfg
        self.tok = Embedding(cfg.vocab_size, cfg.d_model, None, device)
        self.freqs = None                     # radians per position, fp64
        if cfg.rotary_dim:
            if cfg.rotary_dim > cfg.d_model // cfg.n_heads:
                raise TensorError(f"rotary_dim ({cfg.rotary_dim}) exceeds the heads' {cfg.d_model // cfg.n_heads} columns")
            self.freqs = _ops.rotary_frequencies(cfg.rotary_dim, cfg.rotary_base, cfg.rotary_scaling, cfg.rotary_factor, cfg.max_seq, self.tok.weight.t.device)
        else:
            self.pos = Embedding(cfg.max_seq, cfg.d_model, None, device)
        self.blocks: List[DecoderBlock] = [DecoderBlock(cfg, device) for _ in range(cfg.n_layers)]
        self.ln_f = LayerNorm(cfg.d_model, cfg.layer_norm_eps, device)
        self.head = Linear(cfg.d_model, cfg.vocab_size, False, device)

    def name(self): return "decoder_lm"
    def sub_modules(self): return [self.tok, *([] if self.cfg.rotary_dim else [self.pos]), *self.blocks, self.ln_f, self.head]

    def _on_device_change(self, device) -> None:
        if self.freqs is not None:
            self.freqs = self.freqs.to(self.tok.weight.t.device)

    def hidden(self, ids: torch.Tensor, source: Optional[torch.Tensor] = None, source_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`source` [B, Sk, d_model] are another sequence's states and `source_mask` which of them take part, as `ops.cross_attention` takes them."""
        if (source is not None) != self.cfg.cross:
            raise TensorError("a model with cross=True takes a source, one without takes none")
        if source is not None and (source.dim() != 3 or source.shape[0] != ids.shape[0] or source.shape[2] != self.cfg.d_model):
            raise TensorError(f"source must be [{ids.shape[0]}, Sk, {self.cfg.d_model}], not {list(source.shape)}")
        B, S = ids.shape
        x = self.tok.forward(Variable.wrap(ids)).t
        if self.freqs is None:
            x = x + self.pos.forward(Variable.wrap(torch.arange(S, device=ids.device))).t
        if x.is_cuda and _ops.FLAGS.autocast == torch.bfloat16:
            x = x.to(torch.bfloat16)
        if source is not None:
            source = source.to(x.dtype)
        delta = None
        for blk in self.blocks:
            delta, x = blk.forward_pair(delta, x, self.freqs, source, source_mask)
        c = self.cfg
        return _ops.layer_norm(delta, self.ln_f.weight.t, self.ln_f.bias.t, c.layer_norm_eps, residual=x, p_drop=c.dropout,
                               training=self.training)

    def forward(self, ids: Variable, source: Optional[Variable] = None, source_mask: Optional[torch.Tensor] = None) -> Variable:
        return Variable.wrap(_ops.linear(self.hidden(ids.t, None if source is None else source.t, source_mask), self.head.weight.t, None))

    def loss(self, ids: torch.Tensor, targets: torch.Tensor, source: Optional[torch.Tensor] = None, source_mask: Optional[torch.Tensor] = None) -> Variable:
        """Mean next-token cross-entropy; projection + loss fused on CUDA."""
        h = self.hidden(ids, source, source_mask)
        return Variable.wrap(_ops.linear_cross_entropy(h, self.head.weight.t, None, targets.reshape(-1), -100))
