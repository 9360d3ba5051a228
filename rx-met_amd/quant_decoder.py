"""A decoder layer served in 8 bits with the operators of ``decoder_ops``.

``QuantDecoderLayer`` runs attention and feed-forward of one layer on int8 weights (a scale per
output), int8 activations (a scale per token, found at run time) and the paged int8 cache, for
prompts, prompt chunks and single tokens alike::

    layer = QuantDecoderLayer.from_float(norm1, w_qkv, w_o, norm2, w_up, w_down,
                                         heads=32, kv_heads=8)
    cache = KVCache.empty(pages, kv_heads=8, dim=128, page_size=64)
    step = Step(block_table, lengths, cu_new, max_new, max_length)     # of all layers of a pass
    x = layer(x, cache, step)

Positions are the caller's: `rotate`, if given, gets (q, k, positions) after the projection.

With ``QuantExperts`` (from the operators of ``expert_ops``) the feed-forward is one of experts::

    experts = QuantExperts.from_float(w_router, w_up, w_down, top_k=8, gated=True)
    layer = QuantDecoderLayer.from_float(norm1, w_qkv, w_o, norm2, heads=32, kv_heads=8,
                                         experts=experts)
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional

import torch
from torch import nn

import decoder_ops as ops
import expert_ops
from decoder_ops import KVCache  # noqa: F401  (what a layer is called with)


class Step(NamedTuple):
    """Where a pass stands: sequences' pages, the tokens that the cache holds of them before, and
    the rows of x that are theirs (None: one each).  ``max_new`` and ``max_length`` (tokens of a sequence
    after the pass) size the launches; the caller knows them from its schedule."""
    block_table: torch.Tensor
    lengths: torch.Tensor
    cu_new: Optional[torch.Tensor] = None
    max_new: Optional[int] = None
    max_length: Optional[int] = None

    def after(self) -> torch.Tensor:
        """The sequences' lengths once this pass's tokens are in the cache."""
        if self.cu_new is None:
            return self.lengths + 1
        return self.lengths + (self.cu_new[1:] - self.cu_new[:-1])

    def positions(self, tokens: int) -> torch.Tensor:
        """The place of each row of x in its sequence."""
        if self.cu_new is None:
            return self.lengths
        new = (self.cu_new[1:] - self.cu_new[:-1]).long()
        seq = torch.repeat_interleave(torch.arange(len(new), device=new.device), new,
                                      output_size=tokens)
        row = torch.arange(tokens, device=new.device, dtype=torch.int32)
        return self.lengths[seq] + row - self.cu_new[seq]


class QuantExperts(nn.Module):
    """A feed-forward of experts on int8 weights (a scale per output): router, the chosen experts' two
    products, their rows added up.  The logits are float32, from the codes that the experts get.

    The router is in 8 bits like the products, which changes some choices: of random normal tokens and weights
    of width 2048, 1.0 % of the chosen (8 of 64 experts; of width 4096 and 8 of 256 1.5 %), 0.7 % (1.1 %) of it by the
    router's own codes and the rest by the tokens'.  A router that stays in float takes the operators of
    ``expert_ops`` one by one, with its logits for ``route_experts``."""

    def __init__(self, width: int, hidden: int, experts: int, top_k: int, activation: str = "silu",
                 gated: bool = True, score: str = "softmax", with_bias: bool = False, groups: int = 1,
                 top_groups: Optional[int] = None, group_best: int = 1, renormalize: bool = True,
                 scale: float = 1.0, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        super().__init__()
        try:  # what every pass would refuse
            expert_ops._router(experts, top_k, score, groups, top_groups, group_best, renormalize, scale)
        except RuntimeError as e:
            raise ValueError(str(e)) from None
        if activation not in ops.ACTIVATIONS or dtype not in ops._DTYPE:
            raise ValueError(f"experts need an activation of {sorted(a for a in ops.ACTIVATIONS if a)} and "
                             f"dtype float32, float16 or bfloat16, not {activation!r} and {dtype}")
        self.width, self.hidden, self.experts, self.top_k = width, hidden, experts, top_k
        self.activation, self.gated, self.dtype = activation, gated, dtype
        self.choice = dict(score=score, groups=groups, top_groups=top_groups, group_best=group_best,
                           renormalize=renormalize, scale=scale)
        for name, shape in (("router", (experts, width)),
                            ("up", (experts, hidden * (2 if gated else 1), width)),
                            ("down", (experts, width, hidden))):
            self.register_buffer(f"w_{name}", torch.zeros(shape, dtype=torch.int8, device=device))
            self.register_buffer(f"s_{name}", torch.zeros(shape[:-1], dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros(experts, dtype=torch.float32, device=device)
                             if with_bias else None)

    @classmethod
    def from_float(cls, w_router, w_up, w_down, top_k: int, bias=None, gated: bool = True,
                   **kw) -> "QuantExperts":
        """From float weights on the GPU, each row on its own grid: w_router [experts, width], w_up
        [experts, hidden, width] (gated: 2 hidden rows, the gates first), w_down [experts, width,
        hidden]; bias [experts], added to the scores for the choice alone."""
        m = cls(w_router.shape[1], w_down.shape[2], w_router.shape[0], top_k, gated=gated,
                with_bias=bias is not None, device=w_router.device, **kw)
        for name, w in (("router", w_router), ("up", w_up), ("down", w_down)):
            codes, scales = ops.quantize_rows(w.detach())
            if codes.shape != getattr(m, f"w_{name}").shape:
                raise ValueError(f"w_{name} has the shape {tuple(w.shape)}, not "
                                 f"{tuple(getattr(m, f'w_{name}').shape)}")
            getattr(m, f"w_{name}").copy_(codes)
            getattr(m, f"s_{name}").copy_(scales)
        if bias is not None:
            m.bias.copy_(bias.detach())
        return m

    @torch.no_grad()
    def forward(self, codes, scales, residual=None) -> torch.Tensor:
        """codes [tokens, width] with scales [tokens] -> [tokens, width], plus residual."""
        logits = ops.linear_int8(codes, scales, self.w_router, self.s_router, dtype=torch.float32)
        chosen, weights = expert_ops.route_experts(logits, self.top_k, bias=self.bias, **self.choice)
        groups = expert_ops.group_experts(chosen, self.experts)
        u = expert_ops.experts_linear_int8(codes, scales, self.w_up, self.s_up, groups,
                                           activation=self.activation, gated=self.gated,
                                           dtype=self.dtype)
        u, s = ops.quantize_rows(u)
        y = expert_ops.experts_linear_int8(u, s, self.w_down, self.s_down, groups, grouped=True,
                                           dtype=self.dtype)
        return expert_ops.experts_combine(y, weights, groups, residual=residual)


class QuantDecoderLayer(nn.Module):
    """One layer: norm, attention, norm, feed-forward, each with its residual.  The feed-forward is
    two products, or ``experts`` (with ``hidden`` None)."""

    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, hidden: Optional[int],
                 activation: str = "silu", eps: float = 1e-6,
                 dtype: torch.dtype = torch.bfloat16, device="cuda",
                 experts: Optional[QuantExperts] = None):
        super().__init__()
        if (hidden is None) == (experts is None):
            raise ValueError("a layer needs either hidden or experts")
        if experts is not None and (experts.width != width or experts.dtype != dtype):
            raise ValueError(f"experts must have the layer's width and dtype ({width}, {dtype}), not "
                             f"{experts.width} and {experts.dtype}")
        if heads % kv_heads:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        # later it would fail behind the append, with the pass's tokens in the cache
        if dtype not in (torch.float16, torch.bfloat16) or head_dim not in ops.HEAD_DIMS:
            raise ValueError("a layer needs dtype float16 or bfloat16 and a head dimension of "
                             f"{ops.HEAD_DIMS}, not {dtype} and {head_dim}")
        self.width, self.heads, self.kv_heads, self.head_dim = width, heads, kv_heads, head_dim
        self.activation, self.eps, self.dtype = activation, eps, dtype
        qkv = (heads + 2 * kv_heads) * head_dim
        products = [("qkv", qkv, width), ("o", width, heads * head_dim)]
        if experts is None:
            products += [("up", hidden, width), ("down", width, hidden)]
        for name, n, k in products:
            self.register_buffer(f"w_{name}", torch.zeros(n, k, dtype=torch.int8, device=device))
            self.register_buffer(f"s_{name}", torch.zeros(n, dtype=torch.float32, device=device))
        for name in ("norm1", "norm2"):
            self.register_buffer(name, torch.ones(width, dtype=dtype, device=device))
        self.experts = experts

    @classmethod
    def from_float(cls, norm1, w_qkv, w_o, norm2, w_up=None, w_down=None,
                   heads: Optional[int] = None, kv_heads: Optional[int] = None,
                   **kw) -> "QuantDecoderLayer":
        """From float weights [out, in] on the GPU, each row on its own grid; w_up and w_down are left
        out where ``experts`` are given."""
        if heads is None or kv_heads is None:
            raise TypeError("heads and kv_heads are needed")
        if (w_up is None) != (w_down is None) or (w_up is not None and kw.get("experts") is not None):
            raise ValueError("w_up and w_down are needed both, or neither where experts are given")
        width = w_qkv.shape[1]
        layer = cls(width, heads, kv_heads, w_o.shape[1] // heads,
                    None if w_up is None else w_up.shape[0], device=w_qkv.device, **kw)
        products = [("qkv", w_qkv), ("o", w_o)]
        if layer.experts is None:
            products += [("up", w_up), ("down", w_down)]
        for name, w in products:
            codes, scales = ops.quantize_rows(w.detach())
            if codes.shape != getattr(layer, f"w_{name}").shape:
                raise ValueError(f"w_{name} has the shape {tuple(w.shape)}, not "
                                 f"{tuple(getattr(layer, f'w_{name}').shape)}")
            getattr(layer, f"w_{name}").copy_(codes)
            getattr(layer, f"s_{name}").copy_(scales)
        layer.norm1.copy_(norm1.detach())
        layer.norm2.copy_(norm2.detach())
        return layer

    def _linear(self, name, codes, scales, **kw):
        return ops.linear_int8(codes, scales, getattr(self, f"w_{name}"),
                               getattr(self, f"s_{name}"), dtype=self.dtype, **kw)

    @torch.no_grad()
    def forward(self, x, cache: KVCache, step: Step,
                rotate: Optional[Callable] = None) -> torch.Tensor:
        """x [tokens, width] -> the same; the tokens' keys and values go into the cache."""
        n, d = x.shape[0], self.head_dim
        codes, scales, _ = ops.rms_norm_quantize(x, self.norm1, eps=self.eps)
        qkv = self._linear("qkv", codes, scales).view(n, self.heads + 2 * self.kv_heads, d)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        if rotate is not None:
            q, k = rotate(q, k, step.positions(n))
        ops.kv_cache_append(cache, k, v, step.block_table, step.lengths, step.cu_new, step.max_new)
        a = ops.kv_cache_attention(q, cache, step.block_table, step.after(), cu_query=step.cu_new,
                                   max_query=step.max_new, max_length=step.max_length)
        codes, scales = ops.quantize_rows(a.view(n, self.heads * d))
        a = self._linear("o", codes, scales)
        codes, scales, h = ops.rms_norm_quantize(a, self.norm2, x, eps=self.eps)
        if self.experts is not None:
            return self.experts(codes, scales, residual=h)
        codes, scales = ops.quantize_rows(
            self._linear("up", codes, scales, activation=self.activation))
        return self._linear("down", codes, scales, residual=h)
