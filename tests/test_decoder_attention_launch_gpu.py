"""Attention calls whose launch is sized by more rows than the sequences have."""
import pytest
import torch

import decoder_ops as ops

pytestmark = pytest.mark.gpu


def test_many_sequences_without_max_query(cuda):
    """4096 sequences of 20 queries and 8 heads: a tile for each of all rows, for each sequence, would be more
    workgroups than a launch takes.  The same kernel with the sizes given: the same bits."""
    seqs, n, heads, dim = 4096, 20, 8, 64
    g = torch.Generator(device=cuda).manual_seed(0)
    code = lambda *s: torch.randint(-127, 128, s, generator=g, device=cuda).to(torch.int8)
    scale = lambda: torch.rand(seqs, heads, generator=g, device=cuda) / 60 + 1e-3
    cache = ops.KVCache(code(seqs, heads, 32, dim), code(seqs, heads, dim, 32), scale(), scale())
    table = torch.randperm(seqs, generator=g, device=cuda).int()[:, None]
    lengths = torch.full((seqs,), 27, dtype=torch.int32, device=cuda)
    lengths[5] = 20
    cu = torch.arange(seqs + 1, dtype=torch.int32, device=cuda) * n
    q = torch.randn(seqs * n, heads, dim, generator=g, device=cuda).bfloat16()
    out = ops.kv_cache_attention(q, cache, table, lengths, cu)
    assert torch.equal(out, ops.kv_cache_attention(q, cache, table, lengths, cu, max_query=64))
    few = ops.kv_cache_attention(q, cache, table, lengths, cu, max_query=n)  # sixteen rows a workgroup
    assert torch.allclose(out.float(), few.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_one_long_sequence_among_many(cuda):
    """As above, with rows that make a workgroup take several tiles."""
    seqs, heads, dim = 4096, 8, 64
    counts = torch.ones(seqs, dtype=torch.int64)
    counts[7], counts[9] = 90000, 0
    g = torch.Generator(device=cuda).manual_seed(1)
    code = lambda *s: torch.randint(-127, 128, s, generator=g, device=cuda).to(torch.int8)
    ones = torch.full((2, heads), 1 / 60, device=cuda)
    cache = ops.KVCache(code(2, heads, 16, dim), code(2, heads, dim, 16), ones, ones)
    table = torch.zeros(seqs, 1, dtype=torch.int32, device=cuda)
    table[7] = 1
    lengths = torch.full((seqs,), 16, dtype=torch.int32, device=cuda)
    cu = torch.cat([torch.zeros(1), counts.cumsum(0)]).int().to(cuda)
    rows = int(counts.sum())
    q = torch.randn(rows, heads, dim, generator=g, device=cuda).bfloat16()
    out = ops.kv_cache_attention(q, cache, table, lengths, cu, causal=False)
    # the long sequence by itself: its rows in launches of their own
    first = int(counts[:7].sum())
    part = q[first:first + 90000]
    alone = ops.kv_cache_attention(part, cache, table[7:8], lengths[7:8],
                                   torch.tensor([0, 90000], dtype=torch.int32, device=cuda), causal=False)
    assert torch.equal(out[first:first + 90000], alone)
    assert torch.isfinite(out).all()
