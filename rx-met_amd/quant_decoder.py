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
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional

import torch
from torch import nn

import decoder_ops as ops
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


class QuantDecoderLayer(nn.Module):
    """One layer: norm, attention, norm, feed-forward, each with its residual."""

    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, hidden: int,
                 activation: str = "silu", eps: float = 1e-6,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        # later it would fail behind the append, with the pass's tokens in the cache
        if dtype not in (torch.float16, torch.bfloat16) or head_dim not in ops.HEAD_DIMS:
            raise ValueError("a layer needs dtype float16 or bfloat16 and a head dimension of "
                             f"{ops.HEAD_DIMS}, not {dtype} and {head_dim}")
        self.width, self.heads, self.kv_heads, self.head_dim = width, heads, kv_heads, head_dim
        self.activation, self.eps, self.dtype = activation, eps, dtype
        qkv = (heads + 2 * kv_heads) * head_dim
        for name, n, k in (("qkv", qkv, width), ("o", width, heads * head_dim),
                           ("up", hidden, width), ("down", width, hidden)):
            self.register_buffer(f"w_{name}", torch.zeros(n, k, dtype=torch.int8, device=device))
            self.register_buffer(f"s_{name}", torch.zeros(n, dtype=torch.float32, device=device))
        for name in ("norm1", "norm2"):
            self.register_buffer(name, torch.ones(width, dtype=dtype, device=device))

    @classmethod
    def from_float(cls, norm1, w_qkv, w_o, norm2, w_up, w_down, heads: int, kv_heads: int,
                   **kw) -> "QuantDecoderLayer":
        """From float weights [out, in] on the GPU, each row on its own grid."""
        width = w_qkv.shape[1]
        layer = cls(width, heads, kv_heads, w_o.shape[1] // heads, w_up.shape[0],
                    device=w_qkv.device, **kw)
        for name, w in (("qkv", w_qkv), ("o", w_o), ("up", w_up), ("down", w_down)):
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
        codes, scales = ops.quantize_rows(
            self._linear("up", codes, scales, activation=self.activation))
        return self._linear("down", codes, scales, residual=h)
