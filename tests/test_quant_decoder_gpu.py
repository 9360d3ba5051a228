"""A decoder layer in 8 bits on the GPU against the same layer in 64-bit floats, as prompts, as
prompt chunks and token by token."""
import math

import pytest
import torch

import decoder_ops as ops
from quant_decoder import KVCache, QuantDecoderLayer, Step

pytestmark = pytest.mark.gpu

WIDTH, HEADS, KV, DIM, HIDDEN = 256, 4, 2, 64, 640


def weights(cuda, dtype):
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(dtype).to(cuda)
    ones = lambda: (1 + 0.1 * torch.randn(WIDTH, generator=g)).to(dtype).to(cuda)
    return (ones(), rand((HEADS + 2 * KV) * DIM, WIDTH), rand(WIDTH, HEADS * DIM), ones(),
            rand(HIDDEN, WIDTH), rand(WIDTH, HIDDEN))


def float_layer(w, x, lengths):
    """The layer in 64 bits on whole sequences."""
    n1, w_qkv, w_o, n2, w_up, w_down = (t.double().cpu() for t in w)
    norm = lambda v, g: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * g
    out, at = [], 0
    for n in lengths:
        h = x[at:at + n].double().cpu()
        at += n
        qkv = (norm(h, n1) @ w_qkv.t()).view(n, -1, DIM).transpose(0, 1)
        q, k, v = qkv.split((HEADS, KV, KV))
        k, v = k.repeat_interleave(HEADS // KV, 0), v.repeat_interleave(HEADS // KV, 0)
        s = q @ k.transpose(1, 2) / math.sqrt(DIM)
        s = s.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
        a = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, -1)
        h = h + a @ w_o.t()
        u = norm(h, n2) @ w_up.t()
        out.append(h + (u * torch.sigmoid(u)) @ w_down.t())
    return torch.cat(out)


def tables(lengths, page, cuda):
    need = [-(-n // page) for n in lengths]
    t = torch.zeros(len(lengths), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.arange(n) + sum(need[:b])
    return t.to(cuda), sum(need)


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 64])
def test_prompt_chunks_and_tokens(cuda, page, dtype):
    lengths = [70, 33, 5]
    w = weights(cuda, dtype)
    layer = QuantDecoderLayer.from_float(*w, heads=HEADS, kv_heads=KV, dtype=dtype)
    x = torch.randn(sum(lengths), WIDTH, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
    want = float_layer(w, x, lengths)
    table, pages = tables(lengths, page, cuda)
    starts = [0, 70, 103, 108]

    def close(got):
        # Every product's operands are rounded to 127 steps of a row whose largest value is some 3
        # standard deviations: 0.7 % of noise each, against outputs that the residual dominates; four
        # products and the cache leave it below 3 %.
        off = (got.double().cpu() - want).norm() / want.norm()
        assert off < 0.03, off

    # whole prompts
    cache = KVCache.empty(pages, KV, DIM, page, device=cuda)
    step = Step(table, ints([0, 0, 0], cuda), ints(starts, cuda), 70, 70)
    whole = layer(x, cache, step)
    close(whole)
    assert step.after().tolist() == lengths
    assert step.positions(108).tolist() == [i for n in lengths for i in range(n)]

    # in two chunks: the second one's queries see the first one's tokens in the cache
    cache = KVCache.empty(pages, KV, DIM, page, device=cuda)
    first = [40, 20, 0]
    rows, parts, got = [], [first, [n - f for n, f in zip(lengths, first)]], torch.empty_like(x)
    before = [0, 0, 0]
    for new in parts:
        rows = torch.cat([torch.arange(s + b, s + b + n) for s, b, n in zip(starts, before, new)])
        cu = [0, new[0], new[0] + new[1], sum(new)]
        got[rows] = layer(x[rows], cache, Step(table, ints(before, cuda), ints(cu, cuda), max(new), 70))
        before = [b + n for b, n in zip(before, new)]
    close(got)

    # token by token, each sequence for itself
    cache = KVCache.empty(pages, KV, DIM, page, device=cuda)
    for b, n in enumerate(lengths):
        for t in range(n):
            r = starts[b] + t
            got[r:r + 1] = layer(x[r:r + 1], cache, Step(table[b:b + 1], ints([t], cuda), max_length=70))
    close(got)


def test_rotation_gets_positions(cuda):
    w = weights(cuda, torch.bfloat16)
    layer = QuantDecoderLayer.from_float(*w, heads=HEADS, kv_heads=KV)
    cache = KVCache.empty(2, KV, DIM, 64, device=cuda)
    seen = []

    def rotate(q, k, positions):
        seen.append((tuple(q.shape), tuple(k.shape), positions.tolist()))
        return q, k

    x = torch.randn(3, WIDTH, device=cuda).bfloat16()
    layer(x, cache, Step(ints([[0], [1]], cuda), ints([0, 4], cuda), ints([0, 2, 3], cuda), 2, 5), rotate)
    assert seen == [((3, HEADS, DIM), (3, KV, DIM), [0, 1, 4])]


def test_training_form_equals_what_serving_computes(cuda):
    """The fake-quantised norm that a layer is trained with gives the values that the served one's
    codes stand for."""
    x = torch.randn(20, WIDTH, device=cuda).bfloat16()
    r, w = torch.randn_like(x), torch.rand(WIDTH, device=cuda).bfloat16()
    y, h = ops.rms_norm_quantize_dequantize(x, w, r)
    codes, scales, h2 = ops.rms_norm_quantize(x, w, r)
    assert torch.equal(y, (codes * scales[:, None]).bfloat16()) and torch.equal(h, h2)


def test_refusals(cuda):
    with pytest.raises(ValueError, match="multiple"):
        QuantDecoderLayer(64, 3, 2, 64, 128, device=cuda)
    w = list(weights(cuda, torch.bfloat16))
    w[2] = w[2][:100]
    with pytest.raises(ValueError, match="w_o"):
        QuantDecoderLayer.from_float(*w, heads=HEADS, kv_heads=KV)
