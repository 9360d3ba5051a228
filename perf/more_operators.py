"""What the operators of expert layers are measured on.

A feed-forward of experts takes four steps: ``route_experts`` chooses the experts of each token and
weighs them (forward and backward), ``group_experts`` puts the tokens' entries in the experts' order,
``experts_linear_int8`` multiplies each expert's rows of int8 codes with that expert's int8 weight,
with bias, activation and gate, and ``experts_combine`` adds a token's rows up (forward and
backward).

``listed()`` holds named cases from single tokens to long prompts, ``draw()`` gives further ones of
the same ranges.  With ``own`` false, ``run()`` computes a case in elementary torch operations; with
``own`` true it calls the framework.  ``exact()`` is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _ops():
    if os.path.join(_ROOT, "rx-met_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "rx-met_amd"))
    import expert_ops

    return expert_ops


# ----------------------------------------------------------------------------------------------
# The cases
# ----------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of each of 16 sequences: sigmoid scores, a balancing bias, groups of experts
        dict(name="route_decode", kind="route", tokens=16, experts=256, top_k=8, score="sigmoid",
             bias=True, groups=8, top_groups=4, group_best=2, renormalize=True, train=False,
             dtype="float32"),
        # a long prompt through the same router: the choice among 256 counts
        dict(name="route_prompt", kind="route", tokens=16384, experts=256, top_k=8,
             score="sigmoid", bias=True, groups=8, top_groups=4, group_best=2, renormalize=True,
             train=False, dtype="float32"),
        # a training step of a softmax router, weights as they are: all logits get a gradient
        dict(name="route_train", kind="route", tokens=16384, experts=128, top_k=4,
             score="softmax", bias=False, groups=1, top_groups=1, group_best=1, renormalize=False,
             train=True, dtype="bfloat16"),
        # the entries of single tokens in the experts' order: launches count
        dict(name="group_decode", kind="group", tokens=16, experts=256, top_k=8, dropped=0.0),
        # a long prompt's entries; some belong to experts of another process
        dict(name="group_prompt", kind="group", tokens=16384, experts=256, top_k=8, dropped=0.1),
        # single tokens through a gated projection: the weights of the chosen experts count
        dict(name="experts_decode", kind="experts", tokens=16, experts=64, top_k=8, N=1024,
             K=2048, gated=True, grouped=False, bias=False, act="silu", dropped=0.0,
             dtype="bfloat16"),
        # odd sizes in every direction, entries left out, everything that the epilogue does
        dict(name="experts_ragged", kind="experts", tokens=333, experts=13, top_k=3, N=1031,
             K=1025, gated=False, grouped=False, bias=True, act="gelu", dropped=0.2,
             dtype="float16"),
        # a prompt's gated projection, rows gathered from the tokens
        dict(name="experts_up", kind="experts", tokens=8192, experts=32, top_k=8, N=2048, K=2048,
             gated=True, grouped=False, bias=False, act="silu", dropped=0.0, dtype="bfloat16"),
        # its projection back, rows in the experts' order already
        dict(name="experts_down", kind="experts", tokens=8192, experts=32, top_k=8, N=2048,
             K=2048, gated=False, grouped=True, bias=False, act="none", dropped=0.0,
             dtype="bfloat16"),
        # single tokens' rows added up
        dict(name="combine_decode", kind="combine", tokens=16, experts=64, top_k=8, N=2048,
             residual=True, dropped=0.0, train=False, dtype="bfloat16"),
        # a prompt's rows: the rows' bytes count
        dict(name="combine_prompt", kind="combine", tokens=8192, experts=32, top_k=8, N=2048,
             residual=True, dropped=0.0, train=False, dtype="bfloat16"),
        # a training step: the rows' and the weights' gradients too, a width that is odd
        dict(name="combine_train", kind="combine", tokens=8192, experts=32, top_k=8, N=2041,
             residual=True, dropped=0.1, train=True, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    if hi <= lo:
        return lo
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _float(rng):
    return rng.choice(["float32", "float16", "bfloat16", "bfloat16"])


def draw(rng):
    kind = rng.choice(["route", "route", "group", "experts", "experts", "experts", "combine"])
    if kind == "route":
        train = rng.random() < 0.4
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 16 // groups), 1024 // groups)
        tokens = _log(rng, 1, max(1, (1 << (21 if train else 22)) // max(128, experts)))
        best = rng.choice([1, 2])
        top_groups = rng.randint(1, groups)
        top_k = min(_log(rng, 1, 16), top_groups * (experts // groups))
        return dict(kind=kind, tokens=tokens, experts=experts, top_k=top_k,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, group_best=best,
                    renormalize=top_k > 1 and rng.random() < 0.6, train=train, dtype=_float(rng))
    experts = _log(rng, 2, 256)
    top_k = min(experts, rng.choice([1, 2, 2, 3, 4, 6, 8, 8, 10]))
    dropped = rng.choice([0.0, 0.0, 0.1, 0.5])
    if kind == "group":
        return dict(kind=kind, tokens=_log(rng, 4, (1 << 17) // top_k), experts=max(16, experts),
                    top_k=top_k, dropped=dropped)
    if kind == "combine":
        N = _log(rng, 64, 8192)
        return dict(kind=kind, tokens=_log(rng, 1, min(16384, (1 << 27) // (top_k * N))),
                    experts=experts, top_k=top_k, N=N, residual=rng.random() < 0.6,
                    dropped=dropped, train=rng.random() < 0.5, dtype=_float(rng))
    gated = rng.random() < 0.4
    n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
    if rng.random() < 0.6:  # widths of real layers; the others are odd
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    rows = n * (1 + gated)
    experts = min(experts, max(2, (1 << 28) // (rows * k)))
    top_k = min(top_k, experts)
    tokens = (_log(rng, 1, 64) if rng.random() < 0.5
              else _log(rng, 65, max(65, min(8192, (1 << 38) // (rows * k * top_k)))))
    return dict(kind=kind, tokens=tokens, experts=experts, top_k=top_k, N=n, K=k, gated=gated,
                grouped=rng.random() < 0.4, bias=rng.random() < 0.4,
                act=rng.choice(["none", "relu", "silu", "silu", "gelu"]), dropped=dropped,
                dtype=_float(rng))


# ----------------------------------------------------------------------------------------------
# What a program has in hand
# ----------------------------------------------------------------------------------------------

def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)


def _randn_codes(gen, *shape):
    """int8 codes as a normal distribution leaves them on a grid that its largest value spans."""
    half = torch.float16 if math.prod(shape) > (1 << 22) else torch.float32
    return _randn(gen, *shape, dtype=half).mul_(33).round_().clamp_(-127, 127).to(torch.int8)


def _chosen(case, gen):
    """int32 [tokens, top_k]: distinct experts of each token, some more popular than others; -1
    where an entry is left out."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    ids = torch.topk(_randn(gen, T, E) + 0.2 * _randn(gen, E), k, dim=1).indices.to(torch.int32)
    out = torch.randperm(T * k, generator=gen, device=DEV)[:T * k - _kept(case)]
    ids.view(-1)[out] = -1
    return ids


def _kept(case):
    """How many of the tokens' entries belong to an expert."""
    return max(1, round(case["tokens"] * case["top_k"] * (1 - case["dropped"])))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": case}
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if case["kind"] == "group":
        s["experts"] = _chosen(case, gen)
        return s
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "route":
        s["logits"] = (1.5 * _randn(gen, T, E) + 0.5 * _randn(gen, E)).to(dt)
        s["bias"] = 0.05 * _randn(gen, E) if case["bias"] else None
        if case["train"]:
            s["logits"].requires_grad_()
            s["grad"] = 0.1 * _randn(gen, T, k)
        return s
    s["groups"], s["kept"] = _plain_group(_chosen(case, gen), E), _kept(case)
    if case["kind"] == "experts":
        rows, N, K = (T * k if case["grouped"] else T), case["N"], case["K"]
        out = N * (1 + case["gated"])
        s["codes"], s["weight"] = _randn_codes(gen, rows, K), _randn_codes(gen, E, out, K)
        s["scales"] = torch.exp(_randn(gen, rows) * 0.3) / 33
        s["weight_scales"] = torch.exp(_randn(gen, E, out) * 0.3) / (33 * math.sqrt(K))
        s["bias"] = (_randn(gen, E, out) * 0.1).to(dt) if case["bias"] else None
        return s
    s["y"] = _randn(gen, T * k, case["N"]).to(dt)
    w = torch.rand(T, k, generator=gen, device=DEV) + 0.05
    s["weights"] = w / w.sum(1, keepdim=True)
    s["residual"] = _randn(gen, T, case["N"]).to(dt) if case["residual"] else None
    if case["train"]:
        s["grad"] = (0.1 * _randn(gen, T, case["N"])).to(dt)
        for name in ("y", "weights", "residual"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ----------------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"route": _own_route, "group": _own_group, "experts": _own_experts,
                "combine": _own_combine}[kind](s)
    return {"route": _plain_route, "group": lambda s: list(_plain_group(s["experts"], s["case"]["experts"])),
            "experts": _plain_experts, "combine": _plain_combine}[kind](s)


def _own_route(s):
    c = s["case"]
    experts, weights = _ops().route_experts(
        s["logits"], c["top_k"], score=c["score"], bias=s["bias"], groups=c["groups"],
        top_groups=c["top_groups"], group_best=c["group_best"], renormalize=c["renormalize"],
        scale=1.5)
    if not c["train"]:
        return [experts, weights]
    return [experts, weights.detach(), *torch.autograd.grad(weights, s["logits"], s["grad"])]


def _own_group(s):
    return list(_ops().group_experts(s["experts"], s["case"]["experts"]))


def _own_experts(s):
    ops, c = _ops(), s["case"]
    y = ops.experts_linear_int8(s["codes"], s["scales"], s["weight"], s["weight_scales"],
                                ops.ExpertGroups(*s["groups"]), bias=s["bias"],
                                activation=c["act"], gated=c["gated"], grouped=c["grouped"],
                                dtype=_DTYPES[c["dtype"]])
    return y[:s["kept"]]  # the rows behind the experts' last are not written


def _own_combine(s):
    ops, c = _ops(), s["case"]
    out = ops.experts_combine(s["y"], s["weights"], ops.ExpertGroups(*s["groups"]),
                              residual=s["residual"])
    if not c["train"]:
        return out
    inputs = [t for t in (s["y"], s["weights"], s["residual"]) if t is not None]
    return [out.detach(), *torch.autograd.grad(out, inputs, s["grad"])]


# The plain forms: elementary operations, in fp32; scores that a choice goes by in 64 bits, rounded
# to fp32.

def _plain_scores(x, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_route(s):
    c = s["case"]
    T, E, k, G = c["tokens"], c["experts"], c["top_k"], c["groups"]
    logits = s["logits"].detach().float()
    choice = logits
    if c["bias"] or c["group_best"] == 2:
        choice = _plain_scores(logits.double(), c["score"]).float()
        if c["bias"]:
            choice = choice + s["bias"]
    order = choice if c["bias"] else logits
    if G > 1:
        n = min(c["group_best"], E // G)
        value = choice.view(T, G, E // G).sort(dim=-1, descending=True).values[..., :n].sum(-1)
        best = value.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        out = torch.ones(T, G, dtype=torch.bool, device=DEV).scatter_(1, best, False)
        order = torch.where(out.repeat_interleave(E // G, 1), -math.inf, order)
    experts = order.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    score = _plain_scores(logits, c["score"])
    picked = score.gather(1, experts)
    total = picked.sum(-1, keepdim=True) if c["renormalize"] else torch.ones_like(picked[:, :1])
    weights = picked / total
    out = [experts.to(torch.int32), weights * 1.5]
    if c["train"]:
        g = s["grad"] * 1.5
        if c["renormalize"]:
            g = (g - (g * weights).sum(-1, keepdim=True)) / total
        if c["score"] == "sigmoid":
            g = torch.zeros_like(score).scatter_(1, experts, g * picked * (1 - picked))
        else:
            inner = (g * picked).sum(-1, keepdim=True)
            g = torch.zeros_like(score).scatter_(1, experts, g)
            g = score * (g - inner)
        out.append(g.to(s["logits"].dtype))
    return out


def _plain_group(experts, E):
    T, k = experts.shape
    e = experts.reshape(-1).long()
    e = torch.where((e < 0) | (e >= E), E, e)
    ordered, entries = e.sort(stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(E + 1, device=DEV))
    places = torch.empty_like(entries).scatter_(0, entries, torch.arange(T * k, device=DEV))
    places = torch.where(e < E, places, -1)
    return (offsets.to(torch.int32), entries.to(torch.int32), places.view(T, k).to(torch.int32))


def _activate(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain_experts(s):
    c = s["case"]
    offsets, entries, _ = s["groups"]
    E, kept = c["experts"], s["kept"]
    i = torch.arange(kept, device=DEV)
    e = torch.searchsorted(offsets[1:].long(), i, right=True)
    slot = i - offsets.long()[e]
    most = int((offsets[1:] - offsets[:-1]).max())
    row = i if c["grouped"] else entries[:kept].long() // c["top_k"]
    x = torch.zeros(E, max(1, most), c["K"], device=DEV)
    x[e, slot] = s["codes"].float()[row]
    y = torch.bmm(x, s["weight"].float().transpose(1, 2).contiguous())[e, slot]
    y = y * s["scales"][row][:, None] * s["weight_scales"][e]
    if s["bias"] is not None:
        y = y + s["bias"].float()[e]
    if c["gated"]:
        y = _activate(y[:, :c["N"]], c["act"]) * y[:, c["N"]:]
    else:
        y = _activate(y, c["act"])
    return y.to(_DTYPES[c["dtype"]])


def _plain_combine(s):
    c = s["case"]
    T, k, dt = c["tokens"], c["top_k"], _DTYPES[c["dtype"]]
    _, entries, places = s["groups"]
    at, held = places.long().clamp(min=0), (places >= 0)[..., None]
    w = s["weights"].detach()
    rows = torch.where(held, s["y"].detach().float()[at], 0.0)               # [T, k, N]
    out = (rows * w[..., None]).sum(1)
    if s["residual"] is not None:
        out = out + s["residual"].detach().float()
    out = out.to(dt)
    if not c["train"]:
        return out
    g = s["grad"].float()
    dw = (rows * g[:, None]).sum(-1)
    entry = entries.long()
    kept = (torch.arange(T * k, device=DEV) < s["kept"])[:, None]
    dy = torch.where(kept, g[entry // k] * w.reshape(-1)[entry][:, None], 0.0).to(dt)
    return [out, dy, dw] + ([s["grad"].clone()] if s["residual"] is not None else [])


# ----------------------------------------------------------------------------------------------
# Work and the definition in 64 bits
# ----------------------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; products counted as 2 operations."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if case["kind"] == "group":
        return {"bytes": 12 * T * k + 4 * (E + 1), "flops": T * k}
    size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
    if case["kind"] == "route":
        # backward: the logits again, the weights' gradients, and a gradient for every logit
        again = 2 * size * T * E + 8 * T * k if case["train"] else 0
        return {"bytes": size * T * E + 8 * T * k + 4 * E * case["bias"] + again,
                "flops": T * E * (8 + 8 * case["train"])}
    rows = _kept(case)
    N = case["N"]
    if case["kind"] == "combine":
        read = size * N * (rows + T * case["residual"]) + 8 * T * k
        out = size * N * T
        grads = size * N * (2 * rows + T) + 12 * T * k if case["train"] else 0
        return {"bytes": read + out + grads, "flops": N * rows * (6 if case["train"] else 2)}
    out, K = N * (1 + case["gated"]), case["K"]
    used = E * (1 - (1 - k / E) ** (T * (1 - case["dropped"])))  # experts that have rows, about
    read = (T * k if case["grouped"] else T) * (K + 4) + 4 * T * k
    per = out * (K + 4 + size * case["bias"])
    return {"bytes": round(read + used * per + size * rows * N), "flops": 2 * rows * out * K}


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "group": _exact_group, "experts": _exact_experts,
            "combine": _exact_combine}[case["kind"]](s)


def _exact_route(s):
    c = s["case"]
    T, E, G = c["tokens"], c["experts"], c["groups"]
    logits = s["logits"].detach().double().requires_grad_()
    score = torch.special.expit(logits) if c["score"] == "sigmoid" else torch.softmax(logits, -1)
    choice = score.detach().to(torch.float32)  # the choice goes by scores rounded to 32 bits
    if c["bias"]:
        choice = choice.add(s["bias"])
    rank_by = choice.double() if c["bias"] else logits.detach()
    if G > 1:
        members = (choice if c["bias"] or c["group_best"] == 2 else logits.detach().float()).unflatten(1, (G, E // G))
        first, at = members.max(-1, keepdim=True)
        value = first[..., 0]
        if c["group_best"] == 2 and E // G > 1:
            value = value + members.scatter(-1, at, -math.inf).amax(-1)
        # how many groups come before each
        ahead = (value[:, None, :] > value[:, :, None]).sum(-1)
        tie = (value[:, None, :] == value[:, :, None]).tril(-1).sum(-1)
        stays = ahead + tie < c["top_groups"]
        rank_by = rank_by.masked_fill(~stays[..., None].expand(T, G, E // G).flatten(1), -math.inf)
    experts = torch.argsort(-rank_by, dim=1, stable=True)[:, :c["top_k"]]
    weights = torch.take_along_dim(score, experts, 1)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * 1.5
    out = [experts.to(torch.int32), weights.detach()]
    if c["train"]:
        out += torch.autograd.grad(weights, logits, s["grad"].double())
    return out


def _exact_group(s):
    ids, E = s["experts"], s["case"]["experts"]
    members = [[] for _ in range(E + 1)]
    for entry, e in enumerate(ids.flatten().tolist()):
        members[e if 0 <= e < E else E].append(entry)
    offsets, places, entries = [0], [-1] * ids.numel(), []
    for e, held in enumerate(members):
        if e < E:
            for at, entry in enumerate(held):
                places[entry] = offsets[-1] + at
            offsets.append(offsets[-1] + len(held))
        entries += held
    as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    return [as_ints(offsets), as_ints(entries), as_ints(places).view(ids.shape)]


def _exact_experts(s):
    c = s["case"]
    starts = s["groups"][0].tolist()
    row = torch.arange(s["kept"], device=DEV)
    if not c["grouped"]:
        row = torch.div(s["groups"][1][:s["kept"]].long(), c["top_k"], rounding_mode="floor")
    y = torch.empty(s["kept"], c["N"], dtype=torch.float64, device=DEV)
    for e, (a, b) in enumerate(zip(starts, starts[1:])):
        if a == b:
            continue
        v = torch.mm(s["codes"][row[a:b]].double(), s["weight"][e].double().t().contiguous())
        v *= s["scales"][row[a:b]].double()[:, None]
        v *= s["weight_scales"][e].double()
        if s["bias"] is not None:
            v += s["bias"][e].double()
        z = v[:, :c["N"]]
        if c["act"] == "relu":
            z = torch.where(z > 0, z, 0.0)
        elif c["act"] == "silu":
            z = z * torch.special.expit(z)
        elif c["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        y[a:b] = z * v[:, c["N"]:] if c["gated"] else z
    return y


def _exact_combine(s):
    c = s["case"]
    _, _, places = s["groups"]
    T, k, N = c["tokens"], c["top_k"], c["N"]
    y = s["y"].detach().double()
    w = s["weights"].detach().double()
    out = torch.zeros(T, N, dtype=torch.float64, device=DEV)
    if s["residual"] is not None:
        out += s["residual"].detach().double()
    g = s["grad"].double() if c["train"] else None
    dy, dw = torch.zeros_like(y) if c["train"] else None, torch.zeros_like(w)
    for j in range(k):
        t = (places[:, j] >= 0).nonzero()[:, 0]
        p = places[t, j].long()
        out.index_add_(0, t, y[p] * w[t, j, None])
        if c["train"]:
            dy[p] = g[t] * w[t, j, None]
            dw[t, j] = torch.linalg.vecdot(g[t], y[p])
    if not c["train"]:
        return out
    return [out, dy, dw] + ([g] if s["residual"] is not None else [])
