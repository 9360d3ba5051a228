"""What the 8-bit decoder operators are measured on.

A decoder layer that is served in 8 bits runs four operators: the root-mean-square norm that adds
the residual and gives int8 codes with a scale per row (``rms_norm_quantize``, with
``quantize_rows`` where no norm comes before a product and ``rms_norm_quantize_dequantize`` for
training), the int8 matrix product with its epilogue (``linear_int8``), the cache that holds keys
and values as int8 codes with a scale for each page of tokens and head (``kv_cache_append``,
``kv_cache_read``), and the attention over that cache (``kv_cache_attention``).

``listed()`` holds named cases from single tokens to long prompts, ``draw()`` gives further ones of
the same ranges.  With ``own`` false, ``run()`` computes a case in elementary torch operations in
fp32; with ``own`` true it calls the framework.  ``exact()`` is the definition in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-6
_FLOOR = 2.0 ** -112  # least magnitude that a scale is made from


def _ops():
    if os.path.join(_ROOT, "rx-met_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "rx-met_amd"))
    import decoder_ops

    return decoder_ops


# ----------------------------------------------------------------------------------------------
# The cases
# ----------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of each of 16 sequences before a projection: launches and the host count
        dict(name="rms_decode", kind="rms", rows=16, cols=4096, residual=True, norm=True,
             dtype="bfloat16"),
        # a prompt's tokens, with a width that is no multiple of anything
        dict(name="rms_prompt_ragged", kind="rms", rows=3001, cols=4099, residual=True, norm=True,
             dtype="bfloat16"),
        # the input of an output projection, which no norm precedes
        dict(name="rows_prompt", kind="rms", rows=5000, cols=2048, residual=False, norm=False,
             dtype="float16"),
        # a training step's norm, fake-quantised, forward and backward
        dict(name="rms_train", kind="rms_train", rows=8192, cols=4096, residual=True,
             dtype="bfloat16"),
        # a projection of single tokens: the weight's bytes count
        dict(name="linear_decode", kind="linear", M=16, N=4096, K=4096, bias=False, act="none",
             residual=True, dtype="bfloat16"),
        # odd sizes in every direction, with everything that the epilogue does
        dict(name="linear_ragged", kind="linear", M=777, N=2051, K=1025, bias=True, act="gelu",
             residual=True, dtype="float16"),
        # a long prompt's feed-forward product
        dict(name="linear_prompt", kind="linear", M=8192, N=8192, K=8192, bias=True, act="silu",
             residual=False, dtype="bfloat16"),
        # one token for each of 64 sequences goes into its open page, whose codes may be rescaled
        dict(name="append_decode", kind="append", seqs=64, new=1, context=8192, kv_heads=8,
             dim=128, page=64, dtype="bfloat16"),
        # prompts of several lengths, some of them continued
        dict(name="append_prompt", kind="append", seqs=8, new=4096, context=300, kv_heads=8,
             dim=128, page=64, dtype="bfloat16"),
        # two long sequences, one query each: the long axis has to fill the GPU
        dict(name="attn_decode_few", kind="attn", seqs=2, queries=1, context=32768, heads=32,
             kv_heads=8, dim=128, page=64, window=0, dtype="bfloat16"),
        # a full batch of single queries over ragged contexts: the cache's bytes count
        dict(name="attn_decode_many", kind="attn", seqs=64, queries=1, context=16384, heads=64,
             kv_heads=8, dim=128, page=64, window=0, dtype="bfloat16"),
        # prompt chunks over what the cache holds already
        dict(name="attn_prompt", kind="attn", seqs=2, queries=2048, context=6144, heads=32,
             kv_heads=8, dim=128, page=64, window=0, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    if hi <= lo:
        return lo
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rms", "rms_train", "linear", "linear", "append", "attn", "attn", "attn"])
    if kind in ("rms", "rms_train"):
        cols = _log(rng, 64, 16384)
        rows = _log(rng, 1, max(1, min(16384, (1 << 24) // cols)))
        case = dict(kind=kind, rows=rows, cols=cols, residual=rng.random() < 0.6,
                    dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]))
        if kind == "rms":
            case["norm"] = rng.random() < 0.7
            case["residual"] = case["residual"] and case["norm"]
        return case
    if kind == "linear":
        n, k = _log(rng, 64, 12288), _log(rng, 64, 12288)
        if rng.random() < 0.6:  # widths of real layers; the others are odd
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        m = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 65, min(8192, (1 << 39) // (n * k)))
        return dict(kind="linear", M=m, N=n, K=k, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "none", "relu", "silu", "gelu"]),
                    residual=rng.random() < 0.5,
                    dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]))
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    row = kv * dim  # values of one token's key
    if kind == "append":
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        seqs = _log(rng, 1, max(1, min(128, (1 << 25) // (new * row))))
        return dict(kind="append", seqs=seqs, new=new, context=_log(rng, 1, 4096), kv_heads=kv,
                    dim=dim, page=page,
                    dtype=rng.choice(["float32", "float16", "bfloat16", "bfloat16"]))
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    queries = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    context = _log(rng, max(1, queries), 65536 if queries == 1 else 8192)
    most = (1 << 29) // (row * context)
    if queries > 1:
        most = min(most, (1 << 28) // (kv * group * queries * context))
    seqs = _log(rng, 1, max(1, min(64, most)))
    return dict(kind="attn", seqs=seqs, queries=queries, context=context, heads=kv * group,
                kv_heads=kv, dim=dim, page=page,
                window=_log(rng, 1, context) if rng.random() < 0.2 else 0,
                dtype=rng.choice(["float16", "bfloat16"]))


# ----------------------------------------------------------------------------------------------
# What a program has in hand
# ----------------------------------------------------------------------------------------------

def _counts(case):
    """([tokens before], [new tokens or queries]) of the case's sequences: whole numbers that go
    by the case alone.  The first sequence has the most of both; of eight or more one is empty."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    before, new = [], []
    for b in range(case["seqs"]):
        if case["kind"] == "append":
            before.append(case["context"] if b == 0 else rng.randrange(case["context"] + 1))
            new.append(case["new"] if b == 0 else rng.randint((case["new"] + 1) // 2, case["new"]))
        else:
            n = case["queries"] if b == 0 else rng.randint((case["queries"] + 1) // 2,
                                                           case["queries"])
            total = case["context"] if b == 0 else max(n, rng.randint(case["context"] // 4,
                                                                      case["context"]))
            if b == 7:
                total, n = 0, (n if n == 1 else 0)
            before.append(total - n if total else 0)
            new.append(n)
    return before, new


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)


def _randn_codes(gen, *shape):
    """int8 codes as a normal distribution leaves them on a grid that its largest value spans."""
    half = torch.float16 if math.prod(shape) > (1 << 22) else torch.float32
    return _randn(gen, *shape, dtype=half).mul_(33).round_().clamp_(-127, 127).to(torch.int8)


def _cache(case, gen, pages):
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    k, v = _randn_codes(gen, pages, H, P, D), _randn_codes(gen, pages, H, D, P)
    ks = torch.exp(_randn(gen, pages, H) * 0.3) / 33
    vs = torch.exp(_randn(gen, pages, H) * 0.3) / 33
    return k, v, ks, vs


def _table(case, totals, gen):
    """Pages of each sequence in the order that a busy cache hands them out; page 0 stays free."""
    P = case["page"]
    need = [-(-t // P) for t in totals]
    perm = (torch.randperm(max(1, sum(need)), generator=gen, device=DEV) + 1).to(torch.int32)
    table = torch.zeros(len(totals), max(1, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, max(1, sum(need)) + 1


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] in ("rms", "rms_train"):
        r, c = case["rows"], case["cols"]
        # a few channels far above the rest, as the residual stream of a trained model has them
        loud = 1 + 20 * (torch.rand(c, generator=gen, device=DEV) < 0.002).float()
        s["x"] = (_randn(gen, r, c) * loud).to(dt)
        s["residual"] = (_randn(gen, r, c) * loud * 2).to(dt) if case["residual"] else None
        s["weight"] = (1 + 0.2 * _randn(gen, c)).to(dt)
        if case["kind"] == "rms_train":
            s["x"].requires_grad_()
            s["weight"].requires_grad_()
            s["dy"] = (_randn(gen, r, c) * 0.1).to(dt)
            s["dh"] = (_randn(gen, r, c) * 0.1).to(dt)
            if case["residual"]:
                s["residual"].requires_grad_()
        return s
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["codes"], s["weight"] = _randn_codes(gen, M, K), _randn_codes(gen, N, K)
        s["scales"] = torch.exp(_randn(gen, M) * 0.3) / 33
        s["weight_scales"] = torch.exp(_randn(gen, N) * 0.3) / (33 * math.sqrt(K))
        s["bias"] = (_randn(gen, N) * 0.1).to(dt) if case["bias"] else None
        s["residual"] = _randn(gen, M, N).to(dt) if case["residual"] else None
        return s
    before, new = _counts(case)
    totals = [a + n for a, n in zip(before, new)]
    if case["kind"] == "append":
        P = case["page"]
        s["table"], pages = _table(case, totals, gen)
        s["cache"] = _cache(case, gen, pages)
        s["lengths"] = torch.tensor(before, dtype=torch.int32, device=DEV)
        s["cu_new"], s["max_new"] = _starts(new), max(new)
        kv = (_randn(gen, sum(new), 2, case["kv_heads"], case["dim"]) * 1.1).to(dt)
        s["key"], s["value"] = kv[:, 0], kv[:, 1]  # views of one projection's output
        first = [a // P * P for a in before]       # the touched pages' tokens, for the read
        s["first"] = torch.tensor(first, dtype=torch.int32, device=DEV)
        s["cu_read"] = _starts([t - f for t, f in zip(totals, first)])
        s["reads"], s["max_read"] = sum(totals) - sum(first), max(t - f for t, f in zip(totals, first))
        return s
    totals = _totals(case)
    s["table"], pages = _table(case, totals, gen)
    s["cache"] = _cache(case, gen, pages)
    s["lengths"] = torch.tensor(totals, dtype=torch.int32, device=DEV)
    s["cu_query"] = _starts(new) if case["queries"] > 1 else None
    s["max_query"], s["max_length"] = max(new), max(totals)
    s["query"] = (_randn(gen, sum(new), case["heads"], case["dim"]) * 1.5).to(dt)
    return s


def _totals(case):
    """Tokens in the cache of each of an attention case's sequences."""
    before, new = _counts(case)
    return [0 if b == 7 else a + n for b, (a, n) in enumerate(zip(before, new))]


# ----------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"rms": _own_rms, "rms_train": _own_rms_train, "linear": _own_linear,
                "append": _own_append, "attn": _own_attn}[kind](s)
    return {"rms": _plain_rms, "rms_train": _plain_rms_train, "linear": _plain_linear,
            "append": _plain_append, "attn": _plain_attn}[kind](s)


def _own_rms(s):
    ops = _ops()
    if s["case"]["norm"]:
        codes, scales, h = ops.rms_norm_quantize(s["x"], s["weight"], s["residual"], eps=_EPS)
    else:
        codes, scales = ops.quantize_rows(s["x"])
    values = torch.mul(codes, scales[:, None], out=torch.empty_like(s["x"]))  # what the codes stand for
    return [values, scales] + ([h] if s["case"]["norm"] else [])


def _own_rms_train(s):
    ops = _ops()
    y, h = ops.rms_norm_quantize_dequantize(s["x"], s["weight"], s["residual"], eps=_EPS)
    inputs = [t for t in (s["x"], s["weight"], s["residual"]) if t is not None]
    return [y.detach(), h.detach(),
            *torch.autograd.grad([y, h], inputs, [s["dy"], s["dh"]])]


def _own_linear(s):
    return _ops().linear_int8(s["codes"], s["scales"], s["weight"], s["weight_scales"],
                              bias=s["bias"], activation=s["case"]["act"],
                              residual=s["residual"], dtype=_DTYPES[s["case"]["dtype"]])


def _own_append(s):
    ops = _ops()
    cache = ops.KVCache(*s["cache"])
    ops.kv_cache_append(cache, s["key"], s["value"], s["table"], s["lengths"],
                        cu_new=s["cu_new"], max_new=s["max_new"])
    k, v = ops.kv_cache_read(cache, s["table"], s["first"], s["cu_read"], s["reads"],
                             max_tokens=s["max_read"], dtype=s["key"].dtype)
    return [k, v]


def _own_attn(s):
    ops = _ops()
    return ops.kv_cache_attention(s["query"], ops.KVCache(*s["cache"]), s["table"], s["lengths"],
                                  cu_query=s["cu_query"], max_query=s["max_query"],
                                  max_length=s["max_length"],
                                  window=s["case"]["window"] or None)


# The plain forms: fp32, elementary operations.

def _plain_codes(t):
    """(codes as fp32, least scale's magnitude) of the rows of t."""
    top = t.abs().amax(-1, keepdim=True).clamp(min=_FLOOR)
    return torch.round(t * (torch.full_like(top, 127.0) / top)), top


def _plain_rms(s):
    x = s["x"].float()
    if not s["case"]["norm"]:
        codes, top = _plain_codes(x)
        scale = top * (1 / 127)
        return [(codes * scale).to(s["x"].dtype), scale[:, 0]]
    h = x if s["residual"] is None else (x + s["residual"].float()).to(s["x"].dtype).float()
    codes, top = _plain_codes(h * s["weight"].float())
    scale = top * (1 / 127) * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
    return [(codes * scale).to(s["x"].dtype), scale[:, 0], h.to(s["x"].dtype)]


def _plain_rms_train(s):
    dt = s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    h = x
    if s["residual"] is not None:
        h = (x + s["residual"].detach().float()).to(dt).float()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
    codes, top = _plain_codes(h * w)
    y = codes * (top * (1 / 127) * rstd)
    dy, n = s["dy"].float(), h * rstd
    dn = dy * w
    dh = rstd * (dn - n * (dn * n).mean(-1, keepdim=True)) + s["dh"].float()
    dw, dh = (dy * n).sum(0).to(dt), dh.to(dt)
    return [y.to(dt), h.to(dt), dh, dw] + ([dh] if s["residual"] is not None else [])


def _activate(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain_linear(s):
    y = s["codes"].float() @ s["weight"].float().t()
    y = y * s["scales"][:, None] * s["weight_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(_DTYPES[s["case"]["dtype"]])


def _plain_update(pool, scale, ids, x, is_new, is_old, flip):
    """The new tokens x [B, p, H, P, D] go into the pages `ids` [B, p] of the pool; codes that a
    page holds already are rescaled where its scale grows."""
    codes = pool[ids].transpose(-1, -2) if flip else pool[ids]
    old = torch.where(is_old.any(-1)[:, :, None], scale[ids], 0.0)
    top = (x.abs() * is_new[:, :, None, :, None]).amax((-1, -2)).clamp(min=_FLOOR)
    new = torch.maximum(top * (1 / 127), old)
    inv = torch.ones_like(new) / new
    kept = torch.round(codes.float() * (old * inv)[..., None, None])
    put = torch.round(x * inv[..., None, None]).clamp(-127, 127)
    got = torch.where(is_new[:, :, None, :, None], put,
                      torch.where(is_old[:, :, None, :, None], kept, codes.float())).to(torch.int8)
    pool[ids] = got.transpose(-1, -2) if flip else got
    scale[ids] = new


def _plain_append(s):
    k, v, ks, vs = s["cache"]
    P, table, start = s["case"]["page"], s["table"].long(), s["lengths"].long()
    cu = s["cu_new"].long()
    new = cu[1:] - cu[:-1]
    B, pages = len(start), (s["max_new"] + P - 2) // P + 1
    first = start // P
    p = first[:, None] + torch.arange(pages, device=DEV)                     # [B, p]
    touched = p * P < (start + new)[:, None]
    ids = torch.where(touched, table.gather(1, p.clamp(max=table.shape[1] - 1)), 0)
    pos = p[:, :, None] * P + torch.arange(P, device=DEV)                    # [B, p, P]
    is_new = (pos >= start[:, None, None]) & (pos < (start + new)[:, None, None])
    is_old = pos < start[:, None, None]
    at = (cu[:-1, None, None] + pos - start[:, None, None]).clamp(0, s["key"].shape[0] - 1)
    _plain_update(k, ks, ids, s["key"][at].float().transpose(2, 3), is_new, is_old, False)
    _plain_update(v, vs, ids, s["value"][at].float().transpose(2, 3), is_new, is_old, True)
    b = torch.repeat_interleave(torch.arange(B, device=DEV), (s["cu_read"][1:] - s["cu_read"][:-1]).long(),
                                output_size=s["reads"])
    t = s["first"].long()[b] + torch.arange(s["reads"], device=DEV) - s["cu_read"].long()[b]
    page, slot = table[b, t // P], t % P
    dt = s["key"].dtype
    return [(k[page, :, slot].float() * ks[page][..., None]).to(dt),
            (v[page, :, :, slot].float() * vs[page][..., None]).to(dt)]


def _plain_attn(s):
    c = s["case"]
    k, v, ks, vs = s["cache"]
    H, D, P, B = c["kv_heads"], c["dim"], c["page"], c["seqs"]
    G, n, L = c["heads"] // H, s["max_query"], s["max_length"]
    ids = s["table"][:, :-(-L // P)].long()
    keys = (k[ids].float() * ks[ids][..., None, None]).transpose(1, 2).reshape(B, H, -1, D)
    vals = (v[ids].float() * vs[ids][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, H, -1, D)
    length = s["lengths"].long()
    N = s["query"].shape[0]
    if s["cu_query"] is None:
        b = torch.arange(B, device=DEV)
        i, count = torch.zeros_like(b), torch.ones_like(b)
    else:
        cu = s["cu_query"].long()
        count = cu[1:] - cu[:-1]
        b = torch.repeat_interleave(torch.arange(B, device=DEV), count, output_size=N)
        i = torch.arange(N, device=DEV) - cu[b]
    q = torch.zeros(B, n, H, G, D, device=DEV)
    q[b, i] = s["query"].float().view(N, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    score = (q @ keys.transpose(-1, -2) * (1 / math.sqrt(D))).view(B, H, G, n, -1)
    place = (length - count)[:, None] + torch.arange(n, device=DEV)          # [B, n]
    t = torch.arange(keys.shape[2], device=DEV)
    seen = (t <= place[..., None]) & (t < length[:, None, None])
    if c["window"]:
        seen = seen & (t > place[..., None] - c["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    e = torch.where(total > 0, e / total, 0.0)
    out = (e.view(B, H, G * n, -1) @ vals).view(B, H, G, n, D)
    return out.permute(0, 3, 1, 2, 4)[b, i].reshape(N, H * G, D).to(s["query"].dtype)


# ----------------------------------------------------------------------------------------------
# Work and the definition in 64 bits
# ----------------------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; products counted as 2 operations."""
    size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
    if case["kind"] in ("rms", "rms_train"):
        n, c = case["rows"] * case["cols"], case["cols"]
        if case["kind"] == "rms":
            h = 2 * size * n if case["residual"] else 0
            return {"bytes": n * (size + 1) + h + size * c * case["norm"] + 4 * case["rows"],
                    "flops": n * (6 if case["norm"] else 2)}
        # forward: x, residual, h, y; backward: dy, h, dh, dx, and the weight with its gradient
        forward = size * n * (4 if case["residual"] else 2)
        return {"bytes": forward + size * (4 * n + 3 * c), "flops": 20 * n}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 4 * (M + N) + size * (M * N * (1 + case["residual"])
                                                               + N * case["bias"]),
                "flops": 2 * M * N * K}
    before, new = _counts(case)
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        # new tokens in, the touched pages' older tokens in and out, all of them read as values
        old, fresh = sum(a % P for a in before), sum(new)
        return {"bytes": 2 * H * D * (fresh * (size + 1) + 2 * old + (old + fresh) * (1 + size)),
                "flops": 4 * H * D * (old + fresh)}
    held, pairs = 0, 0
    for b, (a, n) in enumerate(zip(before, new)):
        total, w = (0 if b == 7 else a + n), case["window"]
        held += min(total, w + n - 1) if w else total
        seen = [max(0, total - n + i + 1) for i in range(n)]
        pairs += sum(min(t, w) if w else t for t in seen)
    return {"bytes": 2 * H * D * held + 8 * H * -(-held // P)
                     + 2 * size * sum(new) * case["heads"] * D,
            "flops": 4 * case["heads"] * D * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rms": _exact_rms, "rms_train": _exact_rms, "linear": _exact_linear,
            "append": _exact_append, "attn": _exact_attn}[case["kind"]](s)


def _exact_rms(s):
    h = s["x"].detach().double()
    if s["residual"] is not None:
        h = (h + s["residual"].detach().double()).to(s["x"].dtype).double()
    norm = s["case"].get("norm", True)
    w = s["weight"].detach().double() if norm else torch.ones_like(h[0])
    r = torch.sqrt((h.pow(2).sum(1) / h.shape[1] + _EPS).reciprocal()) if norm else torch.ones_like(h[:, 0])
    y = h * r[:, None] * w
    scale = torch.clamp((h * w).abs().max(1).values, min=_FLOOR) * r / 127
    y = (y / scale[:, None]).round() * scale[:, None]
    if s["case"]["kind"] == "rms":
        return [y, scale] + ([h] if norm else [])
    dy, n = s["dy"].double(), h * r[:, None]
    dn = dy * w
    dh = s["dh"].double() + r[:, None] * dn - n * ((dn * n).sum(1) * r / h.shape[1])[:, None]
    dw = torch.einsum("rc,rc->c", dy, n)
    return [y, h, dh, dw] + ([dh] if s["residual"] is not None else [])


def _exact_linear(s):
    y = torch.mm(s["codes"].double(), s["weight"].double().t().contiguous())
    y *= s["scales"].double()[:, None]
    y *= s["weight_scales"].double()[None]
    if s["bias"] is not None:
        y += s["bias"].double()
    act = s["case"]["act"]
    if act == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif act == "silu":
        y = y * torch.special.expit(y)
    elif act == "gelu":
        y = y * torch.special.ndtr(y)
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_append(s):
    P, outs = s["case"]["page"], []
    before, new = _counts(s["case"])
    cu = s["cu_new"].tolist()
    for codes, scale, x, flip in ((s["cache"][0], s["cache"][2], s["key"], False),
                                  (s["cache"][1], s["cache"][3], s["value"], True)):
        parts = []
        for b, (a, n) in enumerate(zip(before, new)):
            fresh = x[cu[b]:cu[b] + n].double()
            tail, ids = a % P, s["table"][b].long()
            full = torch.zeros(-(-(tail + n) // P) * P, *fresh.shape[1:], dtype=torch.float64, device=DEV)
            full[tail:tail + n] = fresh
            pages = full.view(-1, P, *fresh.shape[1:])
            sc = pages.abs().amax((1, 3)).clamp(min=_FLOOR) / 127             # [p, H]
            if tail:
                page = codes[ids[a // P]].double()                            # [H, ., .]
                page = page.transpose(1, 2) if flip else page
                was = scale[ids[a // P]].double()
                sc[0] = torch.maximum(sc[0], was)
                kept = (page * (was / sc[0])[:, None, None]).round() * sc[0][:, None, None]
            vals = (pages / sc[:, None, :, None]).round().clamp(-127, 127) * sc[:, None, :, None]
            vals = vals.reshape(full.shape)
            if tail:
                vals[:tail] = kept.transpose(0, 1)[:tail]
            parts.append(vals[:tail + n])
        outs.append(torch.cat(parts))
    return outs


def _exact_attn(s):
    c = s["case"]
    k, v, ks, vs = s["cache"]
    H, D = c["kv_heads"], c["dim"]
    G, out, at = c["heads"] // H, [], 0
    for total, n, ids in zip(_totals(c), _counts(c)[1], s["table"].long()):
        q = s["query"][at:at + n].double()
        at += n
        res = torch.zeros(n, H, G, D, dtype=torch.float64, device=DEV)
        if total and n:
            page = ids[:-(-total // c["page"])]
            last = torch.arange(total - n, total, device=DEV)[:, None]
            t = torch.arange(total, device=DEV)[None]
            hidden = t > last
            if c["window"]:
                hidden = hidden | (t <= last - c["window"])
            for h in range(H):
                kk = (k[page, h].double() * ks[page, h].double()[:, None, None]).flatten(0, 1)[:total]
                vv = (v[page, h].double() * vs[page, h].double()[:, None, None])
                vv = vv.transpose(1, 2).flatten(0, 1)[:total]
                z = torch.mm(q[:, h * G:(h + 1) * G].flatten(0, 1), kk.t().contiguous()) / math.sqrt(D)
                z = z.view(n, G, total).masked_fill(hidden[:, None], -math.inf)
                res[:, h] = torch.softmax(z, -1) @ vv
        out.append(res.reshape(n, H * G, D))
    return torch.cat(out)
