"""Modules of a decoder-only transformer in PAM arithmetic, made of the operators that a step of one runs next to each other:
layer_norm, linear_act, rotary with the heads' norms, bmm and softmax, gated_linear.  For a training step the optimizer's side is
`pam_amd.optim.clip_grad_norm_` and `pam_amd.optim.Adam`.
"""
import math

import torch

from . import block_ops
from .composites import LayerNorm, softmax
from .pam_ops import bmm, mul

__all__ = ["GatedFeedForward", "Attention", "DecoderBlock"]


def _parameter(*shape, std):
    return torch.nn.Parameter(torch.nn.init.trunc_normal_(torch.empty(shape), std=std, a=-2 * std, b=2 * std))


class GatedFeedForward(torch.nn.Module):
    """x + down(activation(gate(x')) (*) up(x')) with x' = norm(x): one product for gate and up, one for down with the residual."""

    def __init__(self, width, hidden, activation="silu", *, offset=None, approx_bwd=False):
        super().__init__()
        self.kw = dict(offset=offset, approx_bwd=approx_bwd)
        self.activation = activation
        self.norm = LayerNorm(width, **self.kw)
        self.gate_up = _parameter(2 * hidden, width, std=width ** -0.5)
        self.down = _parameter(width, hidden, std=hidden ** -0.5)

    def forward(self, x):
        h = block_ops.gated_linear(self.norm(x), self.gate_up, None, self.activation, **self.kw)
        return block_ops.linear_act(h, self.down, None, None, x, **self.kw)


class Attention(torch.nn.Module):
    """x + out(attention(norm(x))), causal, `kv_heads` keys' and values' heads shared by `heads` queries' heads, queries and keys
    normed per head and rotated.  cache: a dict that keeps keys and values of the tokens so far from call to call."""

    def __init__(self, width, heads, kv_heads, dim, *, offset=None, approx_bwd=False):
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"Attention: {heads} heads do not share {kv_heads}")
        self.kw = dict(offset=offset, approx_bwd=approx_bwd)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.norm = LayerNorm(width, **self.kw)
        self.qkv = _parameter((heads + 2 * kv_heads) * dim, width, std=width ** -0.5)
        self.q_weight, self.k_weight = (torch.nn.Parameter(torch.ones(dim)) for _ in range(2))
        self.out = _parameter(width, heads * dim, std=(heads * dim) ** -0.5)

    def forward(self, x, cos, sin, cache=None):
        batch, tokens, _ = x.shape
        qkv = block_ops.linear_act(self.norm(x), self.qkv, **self.kw).view(batch, tokens, -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 2)
        seen = cache["k"].shape[1] if cache else 0
        if seen + tokens > cos.shape[0]:
            raise ValueError(f"Attention: {seen} tokens in the cache, {tokens} more, and tables of {cos.shape[0]} positions")
        positions = torch.arange(seen, seen + tokens, device=x.device) if seen else None
        q, k = block_ops.rotary(q, k, cos, sin, positions, q_weight=self.q_weight, k_weight=self.k_weight, **self.kw)
        if cache is not None:
            if seen:
                k, v = torch.cat((cache["k"], k), 1), torch.cat((cache["v"], v), 1)
            cache["k"], cache["v"] = k, v

        def by_head(t):                                # [batch, tokens, heads, dim] -> [batch heads, tokens, dim]
            t = t.repeat_interleave(self.heads // t.shape[2], 2)
            return t.transpose(1, 2).reshape(batch * self.heads, -1, self.dim)
        q, k, v = by_head(q), by_head(k), by_head(v)
        scores = bmm(mul(q, self.dim ** -0.5, **self.kw), k.transpose(1, 2), **self.kw)
        if tokens > 1:
            later = torch.ones(tokens, seen + tokens, dtype=torch.bool, device=x.device).triu(seen + 1)
            scores = scores.masked_fill(later, float("-inf"))
        y = bmm(softmax(scores, dim=-1, **self.kw), v, **self.kw)
        y = y.view(batch, self.heads, tokens, self.dim).transpose(1, 2).reshape(batch, tokens, -1)
        return block_ops.linear_act(y, self.out, None, None, x, **self.kw)


class DecoderBlock(torch.nn.Module):
    """Attention, then GatedFeedForward, each behind a norm and on a residual."""

    def __init__(self, width, heads, kv_heads, dim, hidden, activation="silu", *, offset=None, approx_bwd=False):
        super().__init__()
        kw = dict(offset=offset, approx_bwd=approx_bwd)
        self.attention = Attention(width, heads, kv_heads, dim, **kw)
        self.feed_forward = GatedFeedForward(width, hidden, activation, **kw)

    def forward(self, x, cos, sin, cache=None):
        return self.feed_forward(self.attention(x, cos, sin, cache))
