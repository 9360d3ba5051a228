"""The paged int8 cache and the attention over it on the GPU, against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

import decoder_ops as ops
import decoder_oracle as O

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.to(torch.float64).cpu().numpy()


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def fill(cuda, pages, heads, dim, page, seed, spread=0.3):
    """A cache of random codes; scales spread over a log-normal distribution."""
    g = torch.Generator().manual_seed(seed)
    code = lambda *s: torch.randint(-127, 128, s, generator=g).to(torch.int8).to(cuda)
    scale = lambda: torch.exp(torch.randn(pages, heads, generator=g) * spread).to(cuda) / 60
    return ops.KVCache(code(pages, heads, page, dim), code(pages, heads, dim, page), scale(), scale())


def table_for(totals, page, seed, cuda, cols=None):
    """Random distinct pages; the entries that nothing needs are ids that must not be used."""
    need = [-(-t // page) for t in totals]
    cols = cols or max(1, max(need))
    perm = np.random.default_rng(seed).permutation(sum(need) + 3)
    t, at = np.full((len(totals), cols), -5, np.int32), 0
    t[:, 1::2] = 2 ** 31 - 1
    for b, n in enumerate(need):
        t[b, :n] = perm[at:at + n]
        at += n
    return torch.tensor(t, device=cuda), sum(need) + 3


def token_rows(cache, table, b, total):
    """Codes [total, heads, dim] and scales [total, heads] of keys and values, as stored."""
    P = cache.k.shape[2]
    ids = table[b, :-(-total // P)].long()
    k = cache.k[ids].permute(0, 2, 1, 3).flatten(0, 1)[:total]
    v = cache.v[ids].permute(0, 3, 1, 2).flatten(0, 1)[:total]
    rep = lambda s: s[ids].repeat_interleave(P, 0)[:total]
    return k.cpu().numpy(), f64(rep(cache.k_scale)), v.cpu().numpy(), f64(rep(cache.v_scale))


# ---------------------------------------------------------------------------------
# Append and read
# ---------------------------------------------------------------------------------

def check_append(cache, key, value, table, before, new, cu=True, max_new=None):
    """Appends, and compares every page that was touched with the definition; untouched pages
    keep their bytes."""
    cuda = key.device
    old = [t.clone() for t in cache]
    starts = np.concatenate([[0], np.cumsum(new)])
    ops.kv_cache_append(cache, key, value, table, ints(before, cuda),
                        ints(starts, cuda) if cu else None, max_new)
    P, heads = cache.k.shape[2], cache.k.shape[1]
    tab, touched = table.cpu().numpy(), set()
    for x, pool, scales, opool, oscales, flip in (
            (f64(key), cache.k, cache.k_scale, old[0], old[2], False),
            (f64(value), cache.v, cache.v_scale, old[1], old[3], True)):
        pool, opool = pool.cpu().numpy(), opool.cpu().numpy()
        if flip:
            pool, opool = pool.transpose(0, 1, 3, 2), opool.transpose(0, 1, 3, 2)
        scales, oscales = f64(scales), f64(oscales)
        for b, (a, n) in enumerate(zip(before, new)):
            for p in range(a // P, (a + n - 1) // P + 1 if n else a // P):
                page = tab[b, p]
                touched.add(int(page))
                s0, s1 = max(0, a - p * P), min(P, a + n - p * P)
                rows = x[starts[b] + p * P + s0 - a:starts[b] + p * P + s1 - a]
                for h in range(heads):
                    exact, scale = O.append_page(opool[page, h, :s0], oscales[page, h], rows[:, h])
                    got = pool[page, h, :s1].astype(np.int64)
                    if math.isnan(scale):
                        assert math.isnan(scales[page, h]) and (got == 0).all()
                        continue
                    assert abs(scales[page, h] / scale - 1) < 2.0 ** -22
                    # x * (1 / scale): three roundings of fp32 at up to 127
                    differ = got != np.rint(exact)
                    near = np.abs(np.abs(exact - np.floor(exact)) - 0.5) < 1e-4
                    assert (np.abs(got - exact) < 0.5001).all() and not (differ & ~near).any()
                    # what lies behind the new tokens in a piece is not part of the sequence
    rest = [i for i in range(cache.k.shape[0]) if i not in touched]
    for t, o in zip(cache, old):
        assert torch.equal(t[rest].view(torch.uint8), o[rest].view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 3), (32, 128, 1), (64, 128, 2), (128, 192, 1),
                                            (64, 256, 2)])
def test_append(cuda, page, dim, heads, dtype):
    """Ragged prompts behind nothing, behind part of a page, behind whole pages; then single tokens."""
    before = [0, 1, page - 1, page, 2 * page + 5, 3, 0]
    new = [2 * page + 3, 1, 2, page, 1, 0, page]
    totals = [a + n for a, n in zip(before, new)]
    table, pages = table_for([t + 2 for t in totals], page, 1, cuda)
    cache = fill(cuda, pages, heads, dim, page, 2)
    g = torch.Generator().manual_seed(3)
    # some sequences far above the cache's scales, so that older codes move, others below
    loud = torch.repeat_interleave(torch.tensor([1., 8., .01, 1., 20., 1., 1e-3]), torch.tensor(new))
    kv = (torch.randn(sum(new), 2, heads, dim, generator=g) * loud[:, None, None, None]).to(dtype).to(cuda)
    check_append(cache, kv[:, 0], kv[:, 1], table, before, new, max_new=max(new))
    for step in range(2):
        one = (torch.randn(len(new), heads, 2, dim, generator=g) * (1 + 4 * step)).to(dtype).to(cuda)
        check_append(cache, one[:, :, 0], one[:, :, 1], table, [t + step for t in totals],
                     [1] * len(new), cu=False)


def test_append_values_that_are_not_finite(cuda):
    """A NaN or an infinity makes its page and head NaN, and nothing else; zeros stay zeros."""
    table, pages = table_for([70, 70, 70], 64, 1, cuda)
    cache = fill(cuda, pages, 2, 64, 64, 2)
    x = torch.randn(3 * 70, 2, 64, generator=torch.Generator().manual_seed(1)).to(cuda)
    x[3, 0, 5] = float("nan")
    x[70 + 66, 1, 0] = -float("inf")
    x[140:] = 0
    check_append(cache, x, x.clone(), table, [0, 0, 0], [70, 70, 70])
    key, value = ops.kv_cache_read(cache, table, ints([0, 0, 0], cuda), ints([0, 70, 140, 210], cuda),
                                   210, dtype=torch.float32)
    bad = torch.zeros(210, 2, dtype=torch.bool, device=cuda)
    bad[:64, 0] = True
    bad[70 + 64:140, 1] = True
    for t in (key, value):
        assert torch.isnan(t[bad]).all() and torch.isfinite(t[~bad]).all() and (t[140:] == 0).all()
    # a page that is NaN stays NaN, and a later token does not heal it
    check_append(cache, x[200:203], x[200:203], table, [70, 70, 70], [1, 1, 1], cu=False)


def test_append_leaves_out_what_has_no_page(cuda):
    """Ids outside the cache and places past the table write nothing; counts that do not fit the
    rows neither."""
    cache = fill(cuda, 4, 1, 64, 16, 5)
    old = [t.clone() for t in cache]
    table = ints([[-1, 7], [4, 2 ** 31 - 1]], cuda)
    x = torch.randn(64, 1, 64, device=cuda)
    ops.kv_cache_append(cache, x, x, table, ints([0, 0], cuda), ints([0, 32, 64], cuda))
    ops.kv_cache_append(cache, x, x, table, ints([32, 1000], cuda), ints([0, 32, 64], cuda))
    ops.kv_cache_append(cache, x[:2], x[:2], ints([[1, 2], [3, 0]], cuda), ints([-1, 40], cuda))
    ops.kv_cache_append(cache, x, x, ints([[1, 2], [3, 0]], cuda), ints([0, 0], cuda),
                        ints([64, 90, 70], cuda))
    assert all(torch.equal(a, b) for a, b in zip(cache, old))
    # a count beyond the rows is cut to them, a max_new below the count is only slower
    ops.kv_cache_append(cache, x[:20], x[:20], ints([[1, 2]], cuda), ints([0], cuda),
                        ints([0, 32], cuda), max_new=1)
    other = ops.KVCache(*[t.clone() for t in old])
    ops.kv_cache_append(other, x[:20], x[:20], ints([[1, 2]], cuda), ints([0], cuda),
                        ints([0, 20], cuda))
    assert all(torch.equal(a, b) for a, b in zip(cache, other))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 256), (64, 128), (128, 192)])
def test_read(cuda, page, dim, dtype):
    first, count = [0, 5, page, page - 1, 40], [page * 2 + 1, 1, page, 2, 0]
    totals = [f + c for f, c in zip(first, count)]
    table, pages = table_for(totals, page, 1, cuda)
    cache = fill(cuda, pages, 2, dim, page, 7)
    cu = np.concatenate([[0], np.cumsum(count)])
    key, value = ops.kv_cache_read(cache, table, ints(first, cuda), ints(cu, cuda), int(cu[-1]),
                                   max_tokens=max(count), dtype=dtype)
    for b in range(len(first)):
        k, ks, v, vs = token_rows(cache, table, b, totals[b])
        for got, codes, scale in ((key, k, ks), (value, v, vs)):
            want = torch.tensor((codes * scale[..., None])[first[b]:], dtype=torch.float64)
            # code * scale is rounded to fp32 first, then to the type
            want = want.float().to(dtype)
            assert torch.equal(got[cu[b]:cu[b + 1]].cpu(), want)


def test_read_of_what_has_no_page(cuda):
    cache = fill(cuda, 4, 1, 64, 16, 5)
    key, value = ops.kv_cache_read(cache, ints([[1, -1]], cuda), ints([14], cuda), ints([0, 30], cuda), 30)
    for t in (key, value):
        assert torch.isfinite(t[:2]).all() and torch.isnan(t[2:]).all()
    key, value = ops.kv_cache_read(cache, ints([[1, 2]], cuda), ints([-20], cuda), ints([0, 30], cuda), 30)
    for t in (key, value):
        assert torch.isnan(t[:20]).all() and torch.isfinite(t[20:]).all()


def test_round_trip_holds_half_a_step(cuda):
    """Appended values come back within half of their page's step, and an unrounded fp32 ulp."""
    table, pages = table_for([200, 77], 64, 3, cuda)
    cache = fill(cuda, pages, 2, 128, 64, 2)
    x = torch.randn(277, 2, 128, generator=torch.Generator().manual_seed(1)).to(cuda)
    ops.kv_cache_append(cache, x, -x, table, ints([0, 0], cuda), ints([0, 200, 277], cuda), max_new=200)
    key, value = ops.kv_cache_read(cache, table, ints([0, 0], cuda), ints([0, 200, 277], cuda), 277,
                                   dtype=torch.float32)
    step = x.abs().max() / 127
    assert (key - x).abs().max() <= 0.5001 * step and torch.equal(key, -value)


# ---------------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------------

def check_attention(cuda, cache, table, totals, new, q, cu=True, causal=True, window=None, scale=None, **sizes):
    """Every row against the definition; sequences are the rows of `table`."""
    heads, dim = cache.k.shape[1], cache.k.shape[3]
    G, dtype = q.shape[1] // heads, q.dtype
    starts = np.concatenate([[0], np.cumsum(new)])
    out = ops.kv_cache_attention(q, cache, table, ints(totals, cuda),
                                 ints(starts, cuda) if cu else None, causal=causal, window=window,
                                 scale=scale, **sizes)
    assert out.shape == q.shape and out.dtype == dtype
    got, qd = f64(out), f64(q)
    for b, (total, n) in enumerate(zip(totals, new)):
        k, ks, v, vs = token_rows(cache, table, b, total)
        for h in range(heads):
            rows = slice(starts[b], starts[b + 1]), slice(h * G, (h + 1) * G)
            want, off = O.attention(qd[rows], k[:, h], ks[:, h], v[:, h], vs[:, h], total,
                                    1 / math.sqrt(dim) if scale is None else scale, causal, window or 0)
            tol = off + HALF_ULP[dtype] * np.abs(want) + 2.0 ** -24
            most = torch.finfo(dtype).max  # what lies beyond it rounds to an infinity
            with np.errstate(invalid="ignore"):
                fine = np.abs(got[rows] - want) <= tol
                over = (got[rows] == np.sign(want) * np.inf) & (np.abs(want) + tol > most)
            assert (fine | over).all(), (b, h, np.abs(got[rows] - want).max(), off.min())
    return out


def queries(cuda, n, heads, dim, dtype, seed=0, size=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=g) * size).to(dtype).to(cuda)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_single_queries(cuda, dim, page, dtype):
    """Lengths of zero, one, around groups of 64 and pages, and some that many waves share."""
    totals = [0, 1, 15, 16, 17, 63, 64, 65, 128, 300, 1111]
    table, pages = table_for(totals, page, 1, cuda)
    cache = fill(cuda, pages, 2, dim, page, 2)
    q = queries(cuda, len(totals), 6, dim, dtype)
    out = check_attention(cuda, cache, table, totals, [1] * len(totals), q, cu=False)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("group", [1, 2, 3, 7, 16, 17, 40])
def test_head_groups(cuda, group):
    totals = [70, 5, 200]
    table, pages = table_for(totals, 64, 1, cuda)
    cache = fill(cuda, pages, 3, 64, 64, 2)
    q = queries(cuda, 3, 3 * group, 64, torch.float16)
    check_attention(cuda, cache, table, totals, [1, 1, 1], q, cu=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 1), (128, 64, 4), (128, 32, 3), (192, 128, 2),
                                            (256, 64, 5)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 33), (False, None), (False, 50), (True, 1)])
def test_prompts(cuda, dim, page, group, causal, window, dtype):
    """Ragged query counts, none among them, with and without tokens before them."""
    new = [40, 0, 1, 17, 129, 8]
    totals = [40, 10, 1, 100, 200, 8]
    table, pages = table_for(totals, page, 1, cuda)
    cache = fill(cuda, pages, 2, dim, page, 2)
    q = queries(cuda, sum(new), 2 * group, dim, dtype)
    check_attention(cuda, cache, table, totals, new, q, causal=causal, window=window,
                    max_query=max(new), max_length=max(totals))


@pytest.mark.parametrize("dim,page,group", [(64, 64, 9), (128, 16, 8), (128, 128, 16), (256, 64, 8)])
@pytest.mark.parametrize("window", [None, 40])
def test_many_prompts(cuda, dim, page, group, window):
    """As many query rows as fill the GPU: the largest tiles.  Rows of a part of the sequences are
    compared with the definition, all of them with single calls."""
    seqs, new = 130, [33 - b % 5 for b in range(130)]
    totals = [n + 17 * (b % 9) for b, n in enumerate(new)]
    table, pages = table_for(totals, page, 1, cuda)
    cache = fill(cuda, pages, 2, dim, page, 2)
    q = queries(cuda, sum(new), 2 * group, dim, torch.bfloat16)
    starts = np.concatenate([[0], np.cumsum(new)])
    out = ops.kv_cache_attention(q, cache, table, ints(totals, cuda), ints(starts, cuda),
                                 max_query=max(new), max_length=max(totals), window=window)
    for b in (0, 7, 129):
        rows = slice(starts[b], starts[b + 1])
        got = check_attention(cuda, cache, table[b:b + 1], totals[b:b + 1], new[b:b + 1], q[rows],
                              window=window)
        # another tile and other chunks: fp16 weights and bf16 results of both
        assert torch.allclose(out[rows].float(), got.float(), rtol=2.0 ** -7, atol=4e-3 * float(got.float().abs().max()))


def test_queries_before_the_first_token_see_nothing(cuda):
    """More queries than tokens: those that stand before the first token give 0."""
    table, pages = table_for([3], 64, 1, cuda)
    cache = fill(cuda, pages, 1, 64, 64, 2)
    out = check_attention(cuda, cache, table, [3], [9], queries(cuda, 9, 2, 64, torch.float16))
    assert (out[:6] == 0).all() and (out[6:] != 0).any()


@pytest.mark.parametrize("total", [5000, 8197])
def test_long_axis_is_split_and_joined(cuda, total):
    """Few rows and many tokens, with windows that leave most chunks empty; the same bits on every run."""
    totals = [total, 300]
    table, pages = table_for(totals, 64, 1, cuda)
    cache = fill(cuda, pages, 1, 128, 64, 2)
    q = queries(cuda, 2, 4, 128, torch.bfloat16)
    for window in (None, 100, 3000):
        out = check_attention(cuda, cache, table, totals, [1, 1], q, cu=False, window=window)
        again = ops.kv_cache_attention(q, cache, table, ints(totals, cuda), window=window)
        assert torch.equal(out, again)


def test_sizes_that_the_caller_understates(cuda):
    """max_query and max_length below the device's counts cost time, not results."""
    new, totals = [50, 20], [2000, 700]
    table, pages = table_for(totals, 64, 1, cuda)
    cache = fill(cuda, pages, 2, 64, 64, 2)
    q = queries(cuda, 70, 4, 64, torch.float16)
    for max_query, max_length in ((1, 1), (3, 600), (50, 2000), (4000, 100000)):
        check_attention(cuda, cache, table, totals, new, q, max_query=max_query, max_length=max_length)


def test_scales_far_apart(cuda):
    """Pages whose value scales differ by twelve orders of magnitude, in every order."""
    totals = [64 * 9]
    table, pages = table_for(totals, 16, 1, cuda)
    cache = fill(cuda, pages, 1, 64, 16, 2, spread=0.1)
    g = torch.Generator().manual_seed(8)
    cache.v_scale.copy_(10 ** (torch.rand(pages, 1, generator=g) * 12 - 6).to(cuda))
    check_attention(cuda, cache, table, totals, [1], queries(cuda, 1, 8, 64, torch.float16), cu=False)
    small = ops.KVCache(cache.k, cache.v, cache.k_scale, torch.full_like(cache.v_scale, 1e-30))
    q = queries(cuda, 1, 2, 64, torch.bfloat16)
    check_attention(cuda, small, table, totals, [1], q, cu=False)


@pytest.mark.parametrize("group,lift", [(1, 14), (64, 7)])
def test_many_small_weights_beside_a_large_one(cuda, group, lift):
    """One token with the weight 1 and the value 0, and 65535 with 2^-26.5 and 100: what is kept of each is
    2^-11 of itself or 2^-25 of the factor 2^lift that the weights carry; the result is rounded once more."""
    n, w = 65536, 2.0 ** -26.5
    table, pages = table_for([n], 64, 1, cuda)
    k = torch.zeros(pages, 1, 64, 64, dtype=torch.int8, device=cuda)
    k[table[0, 0].long(), 0, 0, 0] = 127
    v = torch.full((pages, 1, 64, 64), 100, dtype=torch.int8, device=cuda)
    v[table[0, 0].long(), 0, :, 0] = 0
    ones = torch.ones(pages, 1, device=cuda)
    q = torch.zeros(1, group, 64, dtype=torch.float16, device=cuda)
    q[:, :, 0] = 1
    out = ops.kv_cache_attention(q, ops.KVCache(k, v, ones, ones), table, ints([n], cuda), max_length=1,
                                 scale=26.5 * math.log(2) / 127)
    want = 100 * (n - 1) * w / (1 + (n - 1) * w)
    tol = want * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -16) + 100 * n * 2.0 ** (-25 - lift)
    assert np.abs(f64(out) - want).max() <= tol


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e30), (torch.bfloat16, 1e-30), (torch.float16, 6e4)])
def test_large_and_small_queries(cuda, dtype, size):
    """Rows outside fp16's range keep their bits; the scale brings the scores back."""
    totals = [100, 33]
    table, pages = table_for(totals, 32, 1, cuda)
    cache = fill(cuda, pages, 1, 64, 32, 2)
    q = queries(cuda, 2, 3, 64, torch.float32, size=size)
    if dtype == torch.float16:
        q = q.clamp(-6e4, 6e4)
    q[0, 1] = 0
    check_attention(cuda, cache, table, totals, [1, 1], q.to(dtype), cu=False, scale=0.1 / size)


@pytest.mark.parametrize("scale", [0.0, -0.2])
@pytest.mark.parametrize("new", [1, 40])
def test_scale_of_zero_and_below(cuda, new, scale):
    """All tokens alike, and the least alike first; partly hidden groups among them."""
    totals = [100, 64]
    table, pages = table_for(totals, 64, 1, cuda)
    cache = fill(cuda, pages, 1, 64, 64, 2)
    q = queries(cuda, 2 * new, 4, 64, torch.float16)
    check_attention(cuda, cache, table, totals, [new, new], q, scale=scale)


def test_not_finite_stays_where_it_is_seen(cuda):
    """NaN pages that the mask hides, NaN in pages and scales that no token has reached, NaN
    queries: only rows that see them become NaN."""
    page, total = 16, 100
    table, pages = table_for([total], page, 1, cuda)
    cache = fill(cuda, pages, 1, 64, page, 2)
    ids = table[0].long().cpu().numpy()
    rest = [p for p in range(pages) if p not in set(ids)]
    cache.k_scale[rest], cache.v_scale[rest] = float("nan"), float("inf")
    hidden = ids[5]  # tokens 80..95
    for scales in (cache.k_scale, cache.v_scale):
        keep = scales[hidden].clone()
        scales[hidden] = float("nan")
        q = queries(cuda, 40, 2, 64, torch.float16)  # stand at 60..99
        out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), ints([0, 40], cuda))
        assert torch.isfinite(out[:20]).all() and torch.isnan(out[20:]).all()
        out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), ints([0, 40], cuda), window=4)
        assert torch.isfinite(out[:20]).all() and torch.isnan(out[20:39]).all()
        assert torch.isfinite(out[39:]).all()  # sees 96..99
        scales[hidden] = keep
    q = queries(cuda, 4, 2, 64, torch.float16)
    q[1, 0, 3], q[2, 1, 0] = float("nan"), float("inf")
    out = ops.kv_cache_attention(q, cache, table, ints([total], cuda), ints([0, 4], cuda))
    bad = torch.zeros(4, 2, dtype=torch.bool, device=cuda)
    bad[1, 0] = bad[2, 1] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()


def test_missing_pages_give_nan(cuda):
    """An id outside the cache, or a length past the table, gives NaN rows for its sequence alone."""
    cache = fill(cuda, 6, 1, 64, 16, 2)
    table = ints([[0, 1, 2], [3, 99, 4], [-2, 5, 1]], cuda)
    q = queries(cuda, 3, 2, 64, torch.float16)
    out = ops.kv_cache_attention(q, cache, table, ints([48, 48, 48], cuda))
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()
    out = ops.kv_cache_attention(q, cache, table[:1].expand(3, 3), ints([48, 49, 5], cuda))
    assert torch.isfinite(out[[0, 2]]).all() and torch.isnan(out[1]).all()


def test_counts_that_do_not_fit_the_rows(cuda):
    """Counts beyond the query rows are cut; sequences that start outside them compute nothing."""
    cache = fill(cuda, 6, 1, 64, 16, 2)
    table = ints([[0, 1, 2], [3, 4, 5]], cuda)
    q = queries(cuda, 5, 2, 64, torch.float16)
    out = ops.kv_cache_attention(q, cache, table, ints([48, 48], cuda), ints([0, 5, 900], cuda))
    want = ops.kv_cache_attention(q, cache, table[:1], ints([48], cuda), ints([0, 5], cuda))
    assert torch.equal(out, want)


def test_strided_queries_and_tables_on_a_side_stream(cuda):
    totals = [100, 300]
    wide, pages = table_for(totals, 64, 1, cuda, cols=9)
    cache = fill(cuda, pages, 2, 128, 64, 2)
    qkv = queries(cuda, 2, 8, 128, torch.bfloat16)
    q, table = qkv[:, 2:6], wide[:, :5]
    first = check_attention(cuda, cache, table, totals, [1, 1], q, cu=False)
    lengths = ints(totals, cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.kv_cache_attention(q.contiguous(), cache, table.contiguous(), lengths)
    side.synchronize()
    assert torch.equal(first, again)


def test_cache_beyond_32_bit_offsets(cuda):
    """A cache of 2.6 GB: pages at its end are written, read and attended to."""
    heads, dim, page, pages = 8, 128, 64, 40000
    cache = ops.KVCache.empty(pages, heads, dim, page, device=cuda)
    total = 200
    table = ints([[pages - 1, 3, pages - 2, pages - 5]], cuda)
    x = torch.randn(total, heads, dim, generator=torch.Generator().manual_seed(1)).to(cuda)
    ops.kv_cache_append(cache, x, x * 0.5, table, ints([0], cuda), ints([0, total], cuda))
    key, value = ops.kv_cache_read(cache, table, ints([0], cuda), ints([0, total], cuda), total,
                                   dtype=torch.float32)
    step = x.abs().max() / 127
    assert (key - x).abs().max() <= 0.5001 * step and (value * 2 - x).abs().max() <= 0.5001 * step
    ids = table[0].long()
    near = ops.KVCache(*[t[ids].contiguous() for t in cache])
    q = queries(cuda, 1, heads, dim, torch.float16)
    a = ops.kv_cache_attention(q, cache, table, ints([total], cuda), max_length=total)
    b = ops.kv_cache_attention(q, near, ints([[0, 1, 2, 3]], cuda), ints([total], cuda), max_length=total)
    assert torch.equal(a, b)


def test_graph_replays(cuda):
    """A decode step captured once: append and attention follow the lengths that the device holds."""
    totals, heads, dim = [130, 70], 2, 128
    table, pages = table_for([t + 8 for t in totals], 64, 1, cuda)
    cache = fill(cuda, pages, heads, dim, 64, 2)
    twin = ops.KVCache(*[t.clone() for t in cache])
    x = torch.randn(2, heads, dim, device=cuda)
    q = queries(cuda, 2, 4, dim, torch.float16)
    lengths, after = ints(totals, cuda), ints([t + 1 for t in totals], cuda)

    def step(c):
        ops.kv_cache_append(c, x, x, table, lengths)
        return ops.kv_cache_attention(q, c, table, after, max_length=256)

    step(ops.KVCache(*[t.clone() for t in cache]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for k in range(4):
        x.copy_(torch.randn(2, heads, dim, generator=torch.Generator().manual_seed(k)))
        lengths.copy_(ints([t + k for t in totals], cuda))
        after.copy_(lengths + 1)
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(cache, twin))


def test_refusals(cuda):
    cache = fill(cuda, 4, 2, 64, 16, 1)
    table, lengths = ints([[0, 1]], cuda), ints([20], cuda)
    q = queries(cuda, 1, 4, 64, torch.float16)
    x = torch.zeros(1, 2, 64, device=cuda)
    att = lambda q=q, c=cache, t=table, n=lengths, **k: ops.kv_cache_attention(q, c, t, n, **k)
    app = lambda k=x, v=x, c=cache, t=table, n=lengths, **kw: ops.kv_cache_append(c, k, v, t, n, **kw)
    for f in (att, app):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f(c=ops.KVCache(*[t.cpu() for t in cache]))
        with pytest.raises(RuntimeError, match="cache.v must"):
            f(c=cache._replace(v=cache.k))
        with pytest.raises(RuntimeError, match="cache.k_scale"):
            f(c=cache._replace(k_scale=cache.k_scale[:3]))
        with pytest.raises(RuntimeError, match="contiguous"):
            f(c=cache._replace(k_scale=cache.k_scale.t().contiguous().t()))
        with pytest.raises(RuntimeError, match="page_size"):
            f(c=cache._replace(k=cache.k[:, :, :8]))
        with pytest.raises(RuntimeError, match="block_table"):
            f(t=table.long())
        with pytest.raises(RuntimeError, match="block_table"):
            f(t=table[0])
        with pytest.raises(RuntimeError, match="lengths"):
            f(n=ints([1, 2], cuda))
        with pytest.raises(RuntimeError, match="lengths"):
            f(n=lengths.cpu())
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        att(q=q.float())
    with pytest.raises(RuntimeError, match="multiple"):
        att(q=queries(cuda, 1, 3, 64, torch.float16))
    with pytest.raises(RuntimeError, match="one query for each"):
        att(q=queries(cuda, 2, 4, 64, torch.float16))
    with pytest.raises(RuntimeError, match="cu_query"):
        att(cu_query=ints([0], cuda))
    with pytest.raises(RuntimeError, match="window"):
        att(window=0)
    with pytest.raises(RuntimeError, match="one token for each"):
        app(k=torch.cat([x, x]), v=torch.cat([x, x]))
    with pytest.raises(RuntimeError, match="key must be"):
        app(k=x[:, :1], v=x[:, :1])
    with pytest.raises(RuntimeError, match="value must have"):
        app(v=x.half())
    with pytest.raises(RuntimeError, match="cu_tokens"):
        ops.kv_cache_read(cache, table, ints([0], cuda), ints([0], cuda), 1)
    with pytest.raises(RuntimeError, match="dim must be one of"):
        ops.KVCache.empty(1, 1, 100, device=cuda)
