"""Operators of a feed-forward of experts over ``include/rxmet_experts.h``.

- ``route_experts``: the experts of each token and their weights, from softmax or sigmoid scores, with a
  balancing bias and groups of experts; differentiable in the logits;
- ``group_experts``: the tokens' entries in the experts' order (``ExpertGroups``);
- ``experts_linear_int8``: product of int8 codes with each expert's int8 weight, with bias, activation
  and gate, as ``decoder_ops.linear_int8`` has it for one weight;
- ``experts_combine``: a token's rows added up by its weights; differentiable.

An entry is one expert of a token: entry ``t * top_k + j`` is token t's j-th.  Places count the
entries in the experts' order.  Every call is queued on PyTorch's current stream and allocates its
outputs and workspace with PyTorch's allocator.  Nothing is synchronised or copied to the host: how many
entries each expert has stays on the device.
The reference has no counterpart; ``quant_decoder.QuantExperts`` runs them together.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

import rxmet_lib as _rx
from decoder_ops import (ACTIVATIONS, LINEAR_K_MAX, _DTYPE, _float_type, _like, _not_traced, _on_gpu,
                         _rows)

EXPERTS_MAX = 1024
TOP_K_MAX = 64
GROUPS_MAX = 64
SCORES = {"softmax": 0, "sigmoid": 1}

_NATIVE = ("rxmet_route_forward", "rxmet_route_backward", "rxmet_group_experts",
           "rxmet_group_experts_workspace_bytes", "rxmet_experts_linear_int8",
           "rxmet_experts_combine", "rxmet_experts_combine_backward", "rxmet_last_error")
_ext = None


def _native():
    """The same calls in C++ (module ``rxmet_torch``, torch_ext/expert_torch.cpp); False where the
    module cannot be imported.  They return None for what needs a copy or has to be refused: that
    is done here."""
    global _ext
    if _ext is None:
        ext = _rx.torch_ext()
        if ext is not None:
            lib = _rx.load()
            ext.bind_experts([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _NATIVE])
        _ext = ext or False
    return _ext


# ---------------------------------------------------------------------------------
# Routing
# ---------------------------------------------------------------------------------

def _router(experts, top_k, score, groups, top_groups, group_best, renormalize, scale):
    """Struct of a router after its checks."""
    if score not in SCORES:
        raise RuntimeError(f"score must be one of {sorted(SCORES)}, not {score!r}")
    if not 1 <= experts <= EXPERTS_MAX:
        raise RuntimeError(f"there must be 1 to {EXPERTS_MAX} experts, not {experts}")
    if not 1 <= groups <= GROUPS_MAX or experts % groups:
        raise RuntimeError(f"groups must be between 1 and {GROUPS_MAX} and divide the {experts} "
                           f"experts, not {groups}")
    if top_groups is None:
        top_groups = groups
    if not 1 <= top_groups <= groups:
        raise RuntimeError(f"top_groups must be between 1 and groups ({groups}), not {top_groups}")
    if group_best not in (1, 2):
        raise RuntimeError(f"group_best must be 1 or 2, not {group_best}")
    if not 1 <= top_k <= min(TOP_K_MAX, top_groups * (experts // groups)):
        raise RuntimeError(f"top_k must be between 1 and {TOP_K_MAX} and at most the "
                           f"{top_groups * (experts // groups)} experts of the chosen groups, not {top_k}")
    return _rx.Router(experts, top_k, SCORES[score], int(bool(renormalize)), groups, top_groups,
                      group_best, scale)


def _route_forward(logits, bias, router):
    code = _DTYPE[logits.dtype]
    l2, stride = _rows(logits)
    shape, dev = (*logits.shape[:-1], router.top_k), logits.device
    experts = torch.empty(shape, dtype=torch.int32, device=dev)
    weights = torch.empty(shape, dtype=torch.float32, device=dev)
    b = None if bias is None else bias.contiguous()
    with torch.cuda.device(dev):
        _rx.call("rxmet_route_forward", ctypes.byref(router), l2.data_ptr(), stride, _rx.ptr(b),
                 experts.data_ptr(), weights.data_ptr(), l2.shape[0], code, _rx.stream_of(dev))
    return experts, weights


class _Route(torch.autograd.Function):
    """``route_experts`` with the weights' gradient; the choice has none."""

    @staticmethod
    def forward(ctx, logits, bias, router):
        experts, weights = _route_forward(logits, bias, router)
        ctx.router = router
        ctx.packed = logits.dtype, logits.device, tuple(logits.shape)
        ctx.save_for_backward(logits, experts)
        ctx.mark_non_differentiable(experts)
        return experts, weights

    @staticmethod
    def backward(ctx, _, d_weights):
        logits, experts = ctx.saved_tensors
        # unpack hooks may hand back other tensors than were packed
        dtype, dev, shape = ctx.packed
        chosen = (*shape[:-1], ctx.router.top_k)
        _like(logits, "the saved logits", dtype, dev, shape)
        _like(experts, "the saved experts", torch.int32, dev, chosen)
        _like(d_weights, "a gradient", torch.float32, dev, chosen)
        l2, stride = _rows(logits)
        experts, d_weights = experts.contiguous(), d_weights.contiguous()
        out = torch.empty(shape, dtype=dtype, device=dev)
        with torch.cuda.device(dev):
            _rx.call("rxmet_route_backward", ctypes.byref(ctx.router), l2.data_ptr(), stride,
                     experts.data_ptr(), d_weights.data_ptr(), out.data_ptr(), l2.shape[0],
                     _DTYPE[dtype], _rx.stream_of(dev))
        return _once("route_experts", out)[0], None, None


def _once(name, *grads):
    """Gradients of a kernel: under create_graph, going through them has to fail, as they have no graph."""
    if not torch.is_grad_enabled():
        return grads
    fail = torch._C._functions.DelayedError(f"{name} cannot be differentiated twice".encode(),
                                            len(grads))
    out = fail(*(None if t is None else t.detach().requires_grad_() for t in grads))
    return out if isinstance(out, tuple) else (out,)


def route_experts(logits, top_k: int, score: str = "softmax", bias=None, groups: int = 1,
                  top_groups: Optional[int] = None, group_best: int = 1, renormalize: bool = True,
                  scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(experts, weights)`` [..., top_k]: the chosen experts (int32, best first) of each row of
    logits [..., E] and their weights (float32).

    Scores s are ``softmax(logits)`` or ``sigmoid(logits)``.  With a ``bias`` [E] (float32, for balance)
    the experts are ordered by ``s.float() + bias`` (the score rounded to float32), without one by
    their logits; ties go to the lowest index, NaN counts as -infinity.  The experts fall into ``groups``
    runs of equal length; a group's value is the sum of its ``group_best`` (1 or 2) largest members, and
    the experts come from the ``top_groups`` groups of the largest values (None: from all).
    Weights are the chosen scores, without the bias, over their sum (``renormalize``), times
    ``scale``.  A softmax row with a NaN or +infinity has NaN weights, a sigmoid one where a NaN is chosen;
    chosen experts whose logits are all -infinity have weights 0.

    logits float32, float16 or bfloat16, up to 2^24 rows, E up to 1024, top_k up to 64.  Differentiable in logits; the
    bias and the choice get no gradient.
    """
    ext = _ext or _native()
    if ext and score in SCORES and not torch._C._are_functorch_transforms_active():
        out = ext.route_experts(logits, top_k, SCORES[score], bias, groups, top_groups, group_best,
                                renormalize, scale)
        if out is not None:
            return out
    _not_traced("route_experts")
    _on_gpu(logits, "logits")
    _float_type(logits, "logits")
    if logits.dim() < 1:
        raise RuntimeError("logits must be [..., experts]")
    E = logits.shape[-1]
    router = _router(E, top_k, score, groups, top_groups, group_best, renormalize, scale)
    if bias is not None:
        _like(bias, "bias", torch.float32, logits.device, (E,))
        bias = bias.detach()
    return _Route.apply(logits, bias, router)


# ---------------------------------------------------------------------------------
# Order by expert
# ---------------------------------------------------------------------------------

class ExpertGroups(NamedTuple):
    """The entries of [..., top_k] chosen experts in the experts' order, int32: expert e has the places
    ``offsets[e]..offsets[e + 1]``; ``entries`` is the entry of each place (behind the experts' last
    stand those of no expert); ``places`` [..., top_k] the place of each entry, -1 for those."""
    offsets: torch.Tensor
    entries: torch.Tensor
    places: torch.Tensor


def group_experts(experts, num_experts: int) -> ExpertGroups:
    """The order of the entries of experts int32 [..., top_k] by expert; entries of an expert keep
    theirs.  Ids outside 0..num_experts - 1 belong to no expert (experts of another process,
    tokens of a padded batch): such entries are multiplied and added up by nothing.  At most 2^26
    entries."""
    ext = _ext or _native()
    if ext:
        out = ext.group_experts(experts, num_experts)
        if out is not None:
            return ExpertGroups(*out)
    _not_traced("group_experts")
    _on_gpu(experts, "experts")
    dev = experts.device
    _like(experts, "experts", torch.int32, dev)
    if experts.dim() < 1 or not 1 <= experts.shape[-1] <= TOP_K_MAX:
        raise RuntimeError(f"experts must be [..., top_k] with top_k between 1 and {TOP_K_MAX}, not "
                           f"{tuple(experts.shape)}")
    if not 1 <= num_experts <= EXPERTS_MAX:
        raise RuntimeError(f"there must be 1 to {EXPERTS_MAX} experts, not {num_experts}")
    e = experts.contiguous()
    n = e.numel()
    out = ExpertGroups(torch.empty(num_experts + 1, dtype=torch.int32, device=dev),
                       torch.empty(n, dtype=torch.int32, device=dev),
                       torch.empty(e.shape, dtype=torch.int32, device=dev))
    size = _rx.load().rxmet_group_experts_workspace_bytes(n, num_experts)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with torch.cuda.device(dev):
        _rx.call("rxmet_group_experts", e.data_ptr(), n, num_experts, out.offsets.data_ptr(),
                 out.entries.data_ptr(), out.places.data_ptr(), _rx.ptr(ws), _rx.stream_of(dev))
    return out


def _groups(groups, dev):
    """(struct, tokens, top_k, the tensors that it points to) of ``groups`` after its checks."""
    offsets, entries, places = groups
    if places.dim() < 1 or not 1 <= places.shape[-1] <= TOP_K_MAX:
        raise RuntimeError(f"groups.places must be [..., top_k] with top_k between 1 and {TOP_K_MAX}, "
                           f"not {tuple(places.shape)}")
    _like(places, "groups.places", torch.int32, dev)
    k, n = places.shape[-1], places.numel()
    _like(entries, "groups.entries", torch.int32, dev, (n,))
    if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= EXPERTS_MAX + 1:
        raise RuntimeError(f"groups.offsets must have 2 to {EXPERTS_MAX + 1} elements, not the shape "
                           f"{tuple(offsets.shape)}")
    _like(offsets, "groups.offsets", torch.int32, dev)
    held = tuple(t.contiguous() for t in groups)
    return (_rx.ExpertGroups(*(t.data_ptr() for t in held), n // k, k, offsets.shape[0] - 1), n // k,
            k, held)


# ---------------------------------------------------------------------------------
# Product
# ---------------------------------------------------------------------------------

def experts_linear_int8(codes, scales, weight, weight_scales, groups: ExpertGroups, bias=None,
                        activation: Optional[str] = None, gated: bool = False,
                        grouped: bool = False, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act((codes[r] @ weight[e].T) * scales[r] * weight_scales[e] + bias[e])`` [entries, N] in
    ``dtype``, a row for each place of ``groups``, e the place's expert.

    codes int8 [tokens, K] with scales float32 [tokens]: the place's token's row is taken; with
    ``grouped`` codes [entries, K] and scales [entries] are in the experts' order already.  weight int8
    [E, N, K] with weight_scales float32 [E, N]; bias [E, N] in ``dtype``.  With ``gated`` they have 2 N
    rows, and a column is ``act(row n) * (row N + n)``.  activation: None, "relu", "silu" or "gelu" (with
    the error function).  For inference: nothing here carries a gradient.
    The sum over K is exact, the rest float32.  K is at most 131071.  Rows behind the experts' last place are
    not written.  Rows that do not start on 16 bytes (K no multiple of 16) are read more slowly.  At most
    2^24 tokens and fewer than 2^26 entries; ceil(N / 128) (gated: / 64) * (entries / 64 + E) is below 2^22.
    """
    ext = _ext or _native()
    if ext and activation in ACTIVATIONS:
        out = ext.experts_linear_int8(codes, scales, weight, weight_scales, *groups, bias,
                                      ACTIVATIONS[activation], gated, grouped, dtype)
        if out is not None:
            return out
    _not_traced("experts_linear_int8")
    _on_gpu(codes, "codes")
    dev = codes.device
    if dtype not in _DTYPE:
        raise RuntimeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or "
                           f"None, not {activation!r}")
    g, tokens, k, held = _groups(groups, dev)
    if codes.dim() != 2 or weight.dim() != 3:
        raise RuntimeError("codes must be [rows, K] and weight [experts, N, K]")
    E, rows, K = weight.shape
    if E != g.experts:
        raise RuntimeError(f"weight must have the {g.experts} experts of groups, not {E}")
    if not 1 <= K <= LINEAR_K_MAX or rows < 1:
        raise RuntimeError(f"weight must have 1 to {LINEAR_K_MAX} columns, not the shape "
                           f"{tuple(weight.shape)}")
    if gated and rows % 2:
        raise RuntimeError(f"a gated weight must have an even number of rows, not {rows}")
    N = rows // 2 if gated else rows
    n = tokens * k if grouped else tokens
    _like(codes, "codes", torch.int8, dev, (n, K))
    _like(scales, "scales", torch.float32, dev, (n,))
    _like(weight, "weight", torch.int8, dev)
    _like(weight_scales, "weight_scales", torch.float32, dev, (E, rows))
    x2, xs = _rows(codes)
    w3 = weight if weight.stride(2) == 1 or K == 1 else weight.contiguous()
    sx, sw = scales.contiguous(), weight_scales.contiguous()
    b = None
    if bias is not None:
        _like(bias, "bias", dtype, dev, (E, rows))
        b = bias.contiguous()
    y = torch.empty(tokens * k, N, dtype=dtype, device=dev)
    with torch.cuda.device(dev):
        _rx.call("rxmet_experts_linear_int8", ctypes.byref(g), int(grouped), x2.data_ptr(), xs,
                 sx.data_ptr(), w3.data_ptr(), w3.stride(1), w3.stride(0), sw.data_ptr(), _rx.ptr(b),
                 y.data_ptr(), N, K, int(gated), ACTIVATIONS[activation], _DTYPE[dtype],
                 _rx.stream_of(dev))
    del held
    return y


# ---------------------------------------------------------------------------------
# Rows added up
# ---------------------------------------------------------------------------------

def _combine(y, weights, groups, residual):
    g, tokens, k, held = _groups(groups, y.device)
    y2, ys = _rows(y)
    N = y2.shape[1]
    w = weights.contiguous()
    lead = groups.places.shape[:-1]
    r2, rs = _rows(residual) if residual is not None else (None, 0)
    out = torch.empty((*lead, N), dtype=y.dtype, device=y.device)
    with torch.cuda.device(y.device):
        _rx.call("rxmet_experts_combine", ctypes.byref(g), y2.data_ptr(), ys, w.data_ptr(),
                 _rx.ptr(r2), rs, out.data_ptr(), N, _DTYPE[y.dtype], _rx.stream_of(y.device))
    del held
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, groups):
        out = _combine(y, weights, groups, residual)
        ctx.has_residual = residual is not None
        ctx.packed = y.dtype, y.device, tuple(y.shape), tuple(weights.shape), tuple(out.shape)
        ctx.experts = groups.offsets.shape[0]
        ctx.save_for_backward(y, weights, *groups)
        return out

    @staticmethod
    def backward(ctx, d_out):
        y, weights, *groups = ctx.saved_tensors
        # unpack hooks may hand back other tensors than were packed
        dtype, dev, y_shape, w_shape, shape = ctx.packed
        _like(y, "the saved y", dtype, dev, y_shape)
        _like(weights, "the saved weights", torch.float32, dev, w_shape)
        _like(groups[0], "the saved offsets", torch.int32, dev, (ctx.experts,))
        _like(groups[2], "the saved places", torch.int32, dev, w_shape)
        _like(d_out, "a gradient", dtype, dev, shape)
        g, _, _, held = _groups(ExpertGroups(*groups), dev)
        y2, ys = _rows(y)
        d2, ds = _rows(d_out)
        w = weights.contiguous()
        need_y, need_w, need_r = ctx.needs_input_grad[:3]
        dy = torch.empty(y_shape, dtype=dtype, device=dev) if need_y else None
        dw = torch.empty(w_shape, dtype=torch.float32, device=dev) if need_w else None
        with torch.cuda.device(dev):
            _rx.call("rxmet_experts_combine_backward", ctypes.byref(g), d2.data_ptr(), ds,
                     y2.data_ptr(), ys, w.data_ptr(), _rx.ptr(dy), _rx.ptr(dw), y_shape[-1],
                     _DTYPE[dtype], _rx.stream_of(dev))
        del held
        dy, dw = _once("experts_combine", dy, dw)
        return dy, dw, d_out if ctx.has_residual and need_r else None, None


def experts_combine(y, weights, groups: ExpertGroups, residual=None) -> torch.Tensor:
    """``sum_j weights[t, j] * y[place of entry (t, j)] + residual[t]`` [..., N], like y.

    y [entries, N] float32, float16 or bfloat16, a row for each place of ``groups``; weights float32
    [..., top_k], shaped like ``groups.places``; residual [..., N] in y's type.  The sum is float32, in the
    order of j, rounded once.  Entries of no expert add nothing; their rows of y are not read.  A caller may take
    further entries away by setting their places to -1 (what exceeds an expert's capacity); no two may share a place.
    At most 2^23 tokens.
    Differentiable in y (0 for the rows of entries without a place), weights and residual.
    """
    ext = _ext or _native()
    if ext and not torch._C._are_functorch_transforms_active():
        out = ext.experts_combine(y, weights, residual, *groups)
        if out is not None:
            return out
    _not_traced("experts_combine")
    _on_gpu(y, "y")
    _float_type(y, "y")
    dev = y.device
    places = groups.places
    if y.dim() != 2 or y.shape[1] < 1 or y.shape[0] != places.numel():
        raise RuntimeError(f"y must be [{places.numel()}, N] with a row for each entry, not "
                           f"{tuple(y.shape)}")
    _like(weights, "weights", torch.float32, dev, places.shape)
    if residual is not None:
        _like(residual, "residual", y.dtype, dev, (*places.shape[:-1], y.shape[1]))
    _groups(groups, dev)
    return _Combine.apply(y, weights, residual, groups)
