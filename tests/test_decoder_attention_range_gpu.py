"""Attention over pages whose scales lie far apart, seen and hidden: every output against the
definition in 64 bits, with a tolerance that is made from what its own row sees alone."""
import math

import numpy as np
import pytest
import torch

import decoder_ops as ops

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = 2.0 ** -119  # about the scale of a page of zeros


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def f64(t):
    return t.to(torch.float64).cpu().numpy()


def codes_cache(cuda, pages, heads, dim, page, seed=0):
    """Random codes, scales of one."""
    g = torch.Generator().manual_seed(seed)
    code = lambda *s: torch.randint(-127, 128, s, generator=g).to(torch.int8).to(cuda)
    ones = lambda: torch.ones(pages, heads, device=cuda)
    return ops.KVCache(code(pages, heads, page, dim), code(pages, heads, dim, page), ones() / 60, ones())


def queries(cuda, n, heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=g) * 1.5).to(dtype).to(cuda)


def check(cuda, cache, table, total, n, q, window=None, **kw):
    """One causal sequence whose last n tokens ask.  What rounding may change: a weight e times its
    scale is kept to 2^-11 of itself or, where that is more, 2^-30 of the row's largest product of the
    two; maxima, exponentials, logarithms and sums in fp32 change 2^-17 of what is added up."""
    out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), ints([0, n], cuda), window=window, **kw)
    P, heads, dim = cache.k.shape[2], cache.k.shape[1], cache.k.shape[3]
    G, got = q.shape[1] // heads, f64(out).reshape(n, heads, -1, dim)
    ids = table[0, :-(-total // P)].long()
    per_token = lambda s: f64(s[ids].repeat_interleave(P, 0)[:total])
    ks, vs = per_token(cache.k_scale), per_token(cache.v_scale)
    place = total - n + np.arange(n)[:, None]
    t = np.arange(total)[None]
    seen = (t <= place) & ((t > place - window) if window else True)
    for h in range(heads):
        k = f64(cache.k[ids, h].flatten(0, 1)[:total])
        v = f64(cache.v[ids, h].transpose(1, 2).flatten(0, 1)[:total])
        for g in range(G):
            # what is hidden does not enter, whatever it holds
            s = np.where(seen, (f64(q[:, h * G + g]) @ k.T) * np.where(np.isfinite(ks[:, h]), ks[:, h], 0)
                         / math.sqrt(dim), -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            p = np.where(seen, e * np.where(np.isfinite(vs[:, h]), vs[:, h], 0), 0)
            l = e.sum(1, keepdims=True)
            want = p @ v / l
            off = np.maximum(2.0 ** -11 * p, 2.0 ** -30 * p.max(1, keepdims=True) * seen) @ np.abs(v) / l
            off += 2.0 ** -17 * (p @ np.abs(v)) / l
            tiny = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -126  # subnormal results
            tol = off + HALF_ULP[q.dtype] * np.abs(want) + tiny
            bad = ~(np.abs(got[:, h, g] - want) <= tol)
            assert not bad.any(), (h, g, bad.sum(), got[:, h, g][bad][:3], want[bad][:3], tol[bad][:3])
    return out


# query rows of a cache head: one, a few (groups of 16 rows), 64 and more (tiles)
ROWS = [(1, 1), (5, 4), (1, 64), (16, 8)]


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("total,zeros", [
    (65, [(64, 65)]), (257, [(256, 257)]), (641, [(640, 641)]),       # one token of zeros, alone in its page
    (640, [(0, 64)]), (640, [(320, 384)]), (640, [(576, 640)]),       # a page of zeros: first, middle, last
    (1300, [(256, 512), (768, 1300)]), (300, [(0, 300)])])
def test_appended_zeros(cuda, total, zeros, n, group):
    """Tokens whose values are zero, as a padding token or a head that gives nothing has them."""
    x = torch.randn(total, 2, 2, 128, generator=torch.Generator().manual_seed(total)).to(cuda).bfloat16()
    x[:, 1] *= 10
    for a, b in zeros:
        x[a:b, 1] = 0
    pages = -(-total // 64)
    cache = ops.KVCache.empty(pages, 2, 128, 64, device=cuda)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    ops.kv_cache_append(cache, x[:, 0], x[:, 1], table, ints([0], cuda), ints([0, total], cuda))
    check(cuda, cache, table, total, n, queries(cuda, n, 2 * group, 128, torch.bfloat16))


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (128, 256)])
@pytest.mark.parametrize("spread", ["tiny and one", "any"])
def test_scales_as_far_apart_as_they_come(cuda, spread, page, dim, n, group):
    """Value scales of 2^-119 beside 1, and any powers from 2^-119 to 2^20, page by page."""
    total = 1111
    pages = -(-total // page)
    cache = codes_cache(cuda, pages, 1, dim, page)
    g = torch.Generator().manual_seed(page)
    if spread == "any":
        scale = torch.exp2(torch.randint(-119, 21, (pages, 1), generator=g).float())
    else:
        scale = torch.where(torch.rand(pages, 1, generator=g) < 0.5, TINY, 1.0)
    cache.v_scale.copy_(scale)
    table = torch.randperm(pages, generator=g).int().to(cuda)[None]
    q = queries(cuda, n, group, dim, torch.bfloat16)
    check(cuda, cache, table, total, n, q)
    check(cuda, cache, table, total, n, q, window=100)


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("group", [1, 8])  # 40 rows: groups of 16; 320: tiles
@pytest.mark.parametrize("loud", [1e3, 1e6, 1e30])
def test_hidden_pages_do_not_matter(cuda, page, group, loud):
    """The pages of a group of 64 tokens get louder; the first queries see the quiet ones alone."""
    total, n = 48, 40  # queries that stand side by side see the first page, or more
    cache = codes_cache(cuda, 3, 2, 64, page)
    cache.v_scale.copy_(torch.tensor([1e-6, loud, loud])[:, None].expand(3, 2))
    table = ints([[0, 1, 2]], cuda)
    check(cuda, cache, table, total, n, queries(cuda, n, 2 * group, 64, torch.bfloat16))


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("value", [float("inf"), 1e38, float("nan")])
def test_pages_before_the_window_may_hold_anything(cuda, value, n, group):
    """Scales that a page left behind, in the same group of 64 tokens as the window."""
    total, window = 64, 10
    cache = codes_cache(cuda, 4, 1, 64, 16)
    cache.v_scale[0], cache.k_scale[0] = value, value  # tokens 0..15; the first query stands at total - n
    q = queries(cuda, n, group, 64, torch.bfloat16)
    out = check(cuda, cache, ints([[0, 1, 2, 3]], cuda), total, n, q, window=window)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("n,group", ROWS)
def test_a_light_loud_page_beside_a_heavy_quiet_one(cuda, n, group):
    """Keys of a page at a score of 100 (base 2) and more above those of one whose values are 2^60
    times as large: the quiet page decides."""
    cache = codes_cache(cuda, 2, 1, 64, 16)
    cache.k.zero_()
    cache.k[0, 0, :, 0], cache.k_scale[:] = 100, 1.0
    cache.v_scale.copy_(torch.tensor([1.0, 2.0 ** 60])[:, None])
    q = torch.zeros(n, group, 64, dtype=torch.bfloat16, device=cuda)
    q[:, :, 0] = 1
    check(cuda, cache, ints([[0, 1]], cuda), 32, n, q)
    out = ops.kv_cache_attention(q, cache, ints([[0, 1]], cuda), ints([32], cuda), ints([0, n], cuda),
                                 scale=math.log(2))
    want = f64(cache.v[0, 0]).mean(1)  # page 1 adds 2^-100 * 2^60 * 127 at most
    assert np.abs(f64(out[-1]) - want).max() <= 2.0 ** -7 * 127


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("total", [100, 5000])
@pytest.mark.parametrize("exponent", [120, -119])
def test_values_at_the_ends_of_the_range(cuda, exponent, total, n, group):
    """Averages near the largest and the least values, whose sums lie beyond fp32."""
    pages = -(-total // 64)
    cache = codes_cache(cuda, pages, 1, 128, 64)
    cache.v.copy_(cache.v.abs().clamp(min=100))  # all of one sign: nothing cancels
    cache.v_scale.fill_(2.0 ** exponent)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    check(cuda, cache, table, total, n, queries(cuda, n, group, 128, torch.bfloat16))


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("dtype,apart,loud", [(torch.bfloat16, 20, 1), (torch.bfloat16, 24, 30),
                                              (torch.bfloat16, 40, 1), (torch.bfloat16, 100, 5),
                                              (torch.float16, 20, 1), (torch.float16, 21, 30)])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_quiet_channels_beside_loud_ones(cuda, page, dim, dtype, apart, loud, n, group):
    """Query channels 2^apart above the others meet key codes of 0: the quiet ones decide."""
    total = 200
    pages = -(-total // page)
    cache = codes_cache(cuda, pages, 1, dim, page)
    cache.k[..., :loud] = 0
    quiet = 2.0 ** -6 if dtype == torch.float16 else 1.0
    cache.k_scale.fill_(1 / 60 / quiet)
    q = queries(cuda, n, group, dim, torch.float32) * quiet
    q[..., :loud] = quiet * 2.0 ** apart
    q[0, 0, :loud] = 0  # a row without them
    check(cuda, cache, torch.arange(pages, dtype=torch.int32, device=cuda)[None], total, n, q.to(dtype))


@pytest.mark.parametrize("n,group", [(1, 1), (16, 8)])
def test_quiet_channels_with_a_scale_below_zero(cuda, n, group):
    """As above, with the least alike first: against the same call with the keys' signs turned."""
    cache = codes_cache(cuda, 4, 1, 128, 64)
    cache.k[..., 0] = 0
    q = queries(cuda, n, group, 128, torch.bfloat16)
    q[..., 0] = 2.0 ** 24
    table, total = ints([[0, 1, 2, 3]], cuda), 256
    out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), ints([0, n], cuda), scale=-128 ** -0.5)
    turned = cache._replace(k=-cache.k)
    assert torch.equal(out, check(cuda, turned, table, total, n, q))


@pytest.mark.parametrize("n,group", [(1, 1), (1, 64)])
@pytest.mark.parametrize("total,heavy", [(1, 0), (300, 0), (300, 200), (300, 299)])
def test_one_heavy_token_is_rounded_once(cuda, total, heavy, n, group):
    """The result is the token's value, whatever its page's scale: the weight adds no rounding of its own.
    Exponential, logarithm, quotient and scale: 2^-18 at most; the result's rounding to fp16."""
    pages = -(-total // 16)
    cache = codes_cache(cuda, pages, 8, 64, 16)
    cache.v_scale.copy_(torch.exp(torch.randn(pages, 8, generator=torch.Generator().manual_seed(heavy)) * 0.5))
    cache.k.zero_()
    cache.k[heavy // 16, :, heavy % 16, 0], cache.k_scale[:] = 127, 1.0
    q = torch.zeros(n, 8 * group, 64, dtype=torch.float16, device=cuda)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), scale=60 * math.log(2) / 127)
    page = heavy // 16
    want = f64(cache.v[page, :, :, heavy % 16]) * f64(cache.v_scale[page])[:, None]
    got = f64(out).reshape(8, group, 64)
    assert (np.abs(got - want[:, None]) <= (2.0 ** -11 + 2.0 ** -18) * np.abs(want[:, None]) + 2.0 ** -25).all()
