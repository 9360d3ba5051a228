"""8-bit operators of a decoder layer over ``include/rxmet_decoder.h``.

Four operators run such a layer on symmetric int8 grids (value = code * scale, codes -127..127):

- ``rms_norm_quantize``: root-mean-square norm of x + residual, given as int8 codes with a scale per
  row; ``quantize_rows`` is the same without the norm, ``rms_norm_quantize_dequantize`` the
  fake-quantised form for training, with a straight-through gradient;
- ``linear_int8``: product of such codes with int8 weights, with bias, activation and residual;
- ``KVCache``, ``kv_cache_append``, ``kv_cache_read``: a paged cache of int8 keys and values with a
  scale for each page and head;
- ``kv_cache_attention``: attention of single queries or prompt chunks over that cache.

Every call is queued on PyTorch's current stream and allocates its outputs and workspace with
PyTorch's allocator.  Nothing is synchronised or copied to the host: sizes that a launch needs
(``max_new``, ``max_query``, ``max_length``) are the caller's, who knows them from its schedule.
The reference has no counterpart; ``quant_decoder.py`` runs them together.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

import rxmet_lib as _rx

ROW_MAX = 65536
LINEAR_K_MAX = 131071
HEAD_DIMS = (64, 128, 192, 256)
PAGE_SIZES = (16, 32, 64, 128)
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3}

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_NATIVE = ("rxmet_rms_quantize_forward", "rxmet_rms_quantize_backward",
           "rxmet_rms_quantize_backward_workspace_bytes", "rxmet_linear_int8",
           "rxmet_linear_int8_workspace_bytes", "rxmet_kv_append", "rxmet_kv_read",
           "rxmet_kv_attention", "rxmet_kv_attention_workspace_bytes", "rxmet_last_error")
_ext = None


def _native():
    """The same calls in C++ (module ``rxmet_torch``, torch_ext/decoder_torch.cpp), which take
    the host 4 - 6 us each instead of 14 - 18; False where the module cannot be imported.  They
    return None (append: False) for what needs a copy or has to be refused: that is done here."""
    global _ext
    if _ext is None:
        ext = _rx.torch_ext()
        if ext is not None:
            lib = _rx.load()
            ext.bind_decoder([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
                              for n in _NATIVE])
        _ext = ext or False
    return _ext


def _not_traced(name):
    """A trace would hold the outputs' allocations without the kernel that fills them."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{name} cannot be traced; rms_norm_quantize_dequantize can")


def _float_type(t, name):
    if t.dtype not in _DTYPE:
        raise RuntimeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return _DTYPE[t.dtype]


def _on_gpu(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on the GPU ({t.device}): these operators have no "
                           "other path")


def _like(t, name, dtype, device, shape=None):
    """Refuses a tensor of another type, device or shape."""
    if t.dtype != dtype or t.device != device:
        raise RuntimeError(f"{name} must be {dtype} on {device}, not {t.dtype} on {t.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")


def _rows(t):
    """(t as [rows, cols] with a dense last axis, row stride); a copy only where no such view
    of t exists."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t, t.stride(0)


# ---------------------------------------------------------------------------------
# Norm and rows to int8
# ---------------------------------------------------------------------------------

def _check_rows(x, weight, residual):
    _on_gpu(x, "x")
    code = _float_type(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= ROW_MAX:
        raise RuntimeError(f"x must have rows of 1 to {ROW_MAX} elements, not the shape "
                           f"{tuple(x.shape)}")
    if weight is not None:
        if weight.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"weight must be {x.dtype} or float32, not {weight.dtype}")
        _like(weight, "weight", weight.dtype, x.device, x.shape[-1:])
    if residual is not None:
        _like(residual, "residual", x.dtype, x.device, x.shape)
    return code


def _row_forward(x, weight, residual, eps, codes, y, keep_rstd):
    """(codes or None, y or None, scales, rstd or None, h)."""
    code = _check_rows(x, weight, residual)
    # (sizes are tensors while a trace records the training form)
    shape, dev = torch.Size(int(n) for n in x.shape), x.device
    x2, xs = _rows(x)
    rows, cols, xs = int(x2.shape[0]), int(x2.shape[1]), int(xs)
    r2, rs = _rows(residual) if residual is not None else (None, 0)
    rs = int(rs)
    w = weight.contiguous() if weight is not None else None
    h = torch.empty(shape, dtype=x.dtype, device=dev) if residual is not None else None
    out = torch.empty(shape, dtype=torch.int8, device=dev) if codes else None
    val = torch.empty(shape, dtype=x.dtype, device=dev) if y else None
    scales = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep_rstd else None
    with torch.cuda.device(dev):
        _rx.call("rxmet_rms_quantize_forward", x2.data_ptr(), xs, _rx.ptr(r2), rs, _rx.ptr(w),
                 int(w is not None and w.dtype == torch.float32), _rx.ptr(h), _rx.ptr(out),
                 _rx.ptr(val), scales.data_ptr(), _rx.ptr(rstd), rows, cols, code, eps,
                 _rx.stream_of(dev))
    return out, val, scales, rstd, x if h is None else h


def rms_norm_quantize(x, weight, residual=None, eps: float = 1e-6
                      ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes, scales, h)``: h = x + residual (rounded to x's type; x itself without a
    residual) and the int8 grid of ``h / sqrt(mean(h^2) + eps) * weight`` for each row.

    x [..., C] float32, float16 or bfloat16; weight [C] of x's type or float32; residual like x.
    codes int8 [..., C], scales float32 [...].  A row with a NaN or an infinity has scale NaN and
    codes 0.  For inference: nothing here carries a gradient, h neither.
    """
    if weight is None:
        raise RuntimeError("rms_norm_quantize needs a weight (quantize_rows has none)")
    ext = _ext or _native()
    if ext:
        out = ext.rms_norm_quantize(x, weight, residual, eps)
        if out is not None:
            return out
    _not_traced("rms_norm_quantize")
    codes, _, scales, _, h = _row_forward(x, weight, residual, eps, True, False, False)
    return codes, scales, h.detach() if h.requires_grad else h


def quantize_rows(x) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)``: the int8 grid of each row of x [..., C] as it is (scale = largest
    magnitude / 127)."""
    ext = _ext or _native()
    if ext:
        out = ext.quantize_rows(x)
        if out is not None:
            return out
    _not_traced("quantize_rows")
    codes, _, scales, _, _ = _row_forward(x, None, None, 0.0, True, False, False)
    return codes, scales


class _RmsQuantDequant(torch.autograd.Function):
    """``rms_norm_quantize_dequantize`` with the rounding's gradient straight through."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        _, y, _, rstd, h = _row_forward(x, weight, residual, eps, False, True, True)
        ctx.has_residual = residual is not None
        ctx.packed = x.dtype, weight.dtype, x.device, tuple(x.shape)
        if residual is None:
            h = h.view_as(h)
        ctx.save_for_backward(h, weight, rstd)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        # unpack hooks may hand back other tensors than were packed
        dtype, weight_dtype, dev, shape = ctx.packed
        _like(h, "the saved h", dtype, dev, shape)
        _like(weight, "the saved weight", weight_dtype, dev, shape[-1:])
        _like(rstd, "the saved rstd", torch.float32, dev, (math.prod(shape[:-1]),))
        for g in (dy, dh):
            if g is not None:
                _like(g, "a gradient", dtype, dev, shape)
        rstd = rstd.contiguous()
        dx, dw = _row_backward(dy, dh, h, weight, rstd, ctx.needs_input_grad[1])
        if torch.is_grad_enabled():
            # create_graph: the kernel's gradients have no graph, so going through them has to fail
            fail = torch._C._functions.DelayedError(
                b"rms_norm_quantize_dequantize cannot be differentiated twice", 2)
            dx, dw = fail(*(None if t is None else t.detach().requires_grad_() for t in (dx, dw)))
        return dx, dw, dx if ctx.has_residual else None, None


def _row_backward(dy, dh, h, weight, rstd, need_dw):
    dev = h.device
    if dy is None:
        dy = torch.zeros_like(h)
    dy2, ds = _rows(dy)
    dh2, hs = _rows(dh) if dh is not None else (None, 0)
    h2, hst = _rows(h)
    rows, cols = h2.shape
    w = weight.contiguous()
    dx = torch.empty(h.shape, dtype=h.dtype, device=dev)
    dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if need_dw else None
    ws = None
    if need_dw:
        size = _rx.load().rxmet_rms_quantize_backward_workspace_bytes(rows, cols)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _rx.call("rxmet_rms_quantize_backward", dy2.data_ptr(), ds, _rx.ptr(dh2), hs,
                 h2.data_ptr(), hst, w.data_ptr(), int(w.dtype == torch.float32), rstd.data_ptr(),
                 dx.data_ptr(), _rx.ptr(dw), rows, cols, _DTYPE[h.dtype], _rx.ptr(ws),
                 _rx.stream_of(dev))
    return dx, dw


def rms_norm_quantize_dequantize(x, weight, residual=None, eps: float = 1e-6
                                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)``: the values that ``rms_norm_quantize``'s codes stand for, in x's type, and h.

    Differentiable in x, weight and residual; the gradient passes the rounding unchanged, as
    ``QuantizeDequantize`` passes it inside its grid (the grid spans the row, so no element is
    clipped).
    """
    if weight is None:
        raise RuntimeError("rms_norm_quantize_dequantize needs a weight")
    ext = _ext or _native()
    # tracing records the Python function, transforms refuse it; a compiled program calls the C++ one
    # between its graphs
    if (ext and torch._C._get_tracing_state() is None
            and not torch._C._are_functorch_transforms_active()):
        out = ext.rms_norm_quantize_dequantize(x, weight, residual, eps)
        if out is not None:
            return out
    return _RmsQuantDequant.apply(x, weight, residual, eps)


# ---------------------------------------------------------------------------------
# Product
# ---------------------------------------------------------------------------------

def linear_int8(codes, scales, weight, weight_scales, bias=None, activation: Optional[str] = None,
                residual=None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``act((codes @ weight.T) * scales * weight_scales + bias) + residual`` in ``dtype``.

    codes int8 [..., K] with scales float32 [...] (from ``rms_norm_quantize`` /
    ``quantize_rows``); weight int8 [N, K] with weight_scales float32 [N]; bias [N] and residual
    [..., N] in ``dtype``.  activation: None, "relu", "silu" or "gelu" (with the error function).
    For inference: bias and residual get no gradient.
    The sum over K is exact, the rest float32.  K is at most 131071.  Rows that do not start on 16 bytes
    (K no multiple of 16) are copied first where there are more than 16 rows of codes.
    """
    ext = _ext or _native()
    if ext and activation in ACTIVATIONS:
        out = ext.linear_int8(codes, scales, weight, weight_scales, bias, ACTIVATIONS[activation],
                              residual, dtype)
        if out is not None:
            return out
    _not_traced("linear_int8")
    _on_gpu(codes, "codes")
    dev = codes.device
    if dtype not in _DTYPE:
        raise RuntimeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or "
                           f"None, not {activation!r}")
    if codes.dim() < 1 or weight.dim() != 2:
        raise RuntimeError("codes must be [..., K] and weight [N, K]")
    N, K = weight.shape
    if not 1 <= K <= LINEAR_K_MAX or N < 1:
        raise RuntimeError(f"weight must have 1 to {LINEAR_K_MAX} columns, not the shape "
                           f"{tuple(weight.shape)}")
    lead = codes.shape[:-1]
    _like(codes, "codes", torch.int8, dev, (*lead, K))
    _like(scales, "scales", torch.float32, dev, lead)
    _like(weight, "weight", torch.int8, dev)
    _like(weight_scales, "weight_scales", torch.float32, dev, (N,))
    x2, xs = _rows(codes)
    w2, wst = _rows(weight)
    M = x2.shape[0]
    sx, sw = scales.contiguous(), weight_scales.contiguous()
    b = None
    if bias is not None:
        _like(bias, "bias", dtype, dev, (N,))
        b = bias.contiguous()
    r2, rs = None, 0
    if residual is not None:
        _like(residual, "residual", dtype, dev, (*lead, N))
        r2, rs = _rows(residual)
    y = torch.empty((*lead, N), dtype=dtype, device=dev)
    size = _rx.load().rxmet_linear_int8_workspace_bytes(x2.data_ptr(), xs, w2.data_ptr(),
                                                           wst, M, N, K)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with torch.cuda.device(dev):
        _rx.call("rxmet_linear_int8", x2.data_ptr(), xs, sx.data_ptr(), w2.data_ptr(), wst,
                 sw.data_ptr(), _rx.ptr(b), _rx.ptr(r2), rs, y.data_ptr(), M, N, K,
                 ACTIVATIONS[activation], _DTYPE[dtype], _rx.ptr(ws), _rx.stream_of(dev))
    return y


# ---------------------------------------------------------------------------------
# Cache
# ---------------------------------------------------------------------------------

class KVCache(NamedTuple):
    """Pages of int8 keys and values: k [pages, heads, page_size, dim], v [pages, heads, dim,
    page_size] (each dimension's tokens side by side), and their float32 scales [pages, heads]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, page_size: int = 64, device="cuda"
              ) -> "KVCache":
        """A cache of `pages` pages; nothing in it is read before it is appended."""
        if dim not in HEAD_DIMS or page_size not in PAGE_SIZES:
            raise RuntimeError(f"dim must be one of {HEAD_DIMS} and page_size one of "
                               f"{PAGE_SIZES}, not {dim} and {page_size}")
        return cls(torch.empty(pages, heads, page_size, dim, dtype=torch.int8, device=device),
                   torch.empty(pages, heads, dim, page_size, dtype=torch.int8, device=device),
                   torch.empty(pages, heads, dtype=torch.float32, device=device),
                   torch.empty(pages, heads, dtype=torch.float32, device=device))


def _cache_args(cache, block_table, *int_vectors):
    """(struct of the cache, struct of the table, device) after the checks that need no device
    data; int_vectors: (name, tensor or None, length or None) of int32 vectors."""
    k, v, ks, vs = cache
    _on_gpu(k, "the cache")
    dev = k.device
    if k.dim() != 4:
        raise RuntimeError(f"cache.k must be [pages, heads, page_size, dim], not {tuple(k.shape)}")
    pages, heads, P, D = k.shape
    if D not in HEAD_DIMS or P not in PAGE_SIZES or pages < 1 or heads < 1:
        raise RuntimeError(f"cache.k must be [pages, heads, page_size, dim] with page_size in "
                           f"{PAGE_SIZES} and dim in {HEAD_DIMS}, not {tuple(k.shape)}")
    _like(k, "cache.k", torch.int8, dev)
    _like(v, "cache.v", torch.int8, dev, (pages, heads, D, P))
    _like(ks, "cache.k_scale", torch.float32, dev, (pages, heads))
    _like(vs, "cache.v_scale", torch.float32, dev, (pages, heads))
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise RuntimeError("the cache's tensors must be contiguous")
    if block_table.dim() != 2 or block_table.shape[1] < 1:
        raise RuntimeError("block_table must be [sequences, pages], not the shape "
                           f"{tuple(block_table.shape)}")
    _like(block_table, "block_table", torch.int32, dev)
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise RuntimeError("block_table's rows must be dense")
    for name, t, length in int_vectors:
        if t is not None:
            _like(t, name, torch.int32, dev, (length,))
            if not t.is_contiguous():
                raise RuntimeError(f"{name} must be contiguous")
    return (_rx.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, P, D, 0),
            _rx.KvTable(block_table.data_ptr(), block_table.stride(0), *block_table.shape), dev)


def _tokens(t, name, dev, heads, dim):
    """t [tokens, heads, dim] with a dense last axis."""
    if t.dim() != 3 or t.shape[1:] != (heads, dim):
        raise RuntimeError(f"{name} must be [tokens, {heads}, {dim}], not {tuple(t.shape)}")
    if t.device != dev:
        raise RuntimeError(f"{name} must be on {dev}, not on {t.device}")
    return t if t.stride(2) == 1 else t.contiguous()


def kv_cache_append(cache: KVCache, key, value, block_table, lengths, cu_new=None,
                    max_new: Optional[int] = None) -> None:
    """Puts new tokens behind the ``lengths[b]`` tokens that each sequence has in the cache.

    key, value [tokens, heads, dim] float32, float16 or bfloat16 (any strides of the first two
    axes): rows ``cu_new[b]..cu_new[b + 1]`` are sequence b's; without ``cu_new`` there is one
    row for each sequence.  ``max_new``: the most rows of a sequence (default: all rows).
    block_table int32 [sequences, pages]; lengths int32 [sequences], cu_new int32 [sequences + 1]
    on the GPU.  ``lengths`` stays as it is.

    A page that receives tokens has the scale max(its largest new magnitude / 127, its scale if it
    held tokens of the sequence before); where that grows, its older codes are moved to the new
    grid.  The sequences' open pages must be their own.  Tokens whose page is missing (an id outside the cache,
    a place past the table) are left out.
    """
    ext = _ext or _native()
    if ext and ext.kv_append(*cache, key, value, block_table, lengths, cu_new, max_new):
        return
    _not_traced("kv_cache_append")
    seqs = block_table.shape[0] if block_table.dim() else 0
    c, t, dev = _cache_args(cache, block_table, ("lengths", lengths, seqs),
                            ("cu_new", cu_new, seqs + 1))
    code = _float_type(key, "key")
    if value.dtype != key.dtype or value.shape != key.shape:
        raise RuntimeError("value must have key's type and shape")
    key = _tokens(key, "key", dev, c.heads, c.dim)
    value = _tokens(value, "value", dev, c.heads, c.dim)
    n = key.shape[0]
    if cu_new is None:
        if n != seqs:
            raise RuntimeError(f"without cu_new there must be one token for each of the {seqs} "
                               f"sequences, not {n}")
        max_new = 1
    with torch.cuda.device(dev):
        _rx.call("rxmet_kv_append", ctypes.byref(c), ctypes.byref(t), lengths.data_ptr(),
                 _rx.ptr(cu_new), n, n if max_new is None else max_new, key.data_ptr(),
                 key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
                 code, _rx.stream_of(dev))


def kv_cache_read(cache: KVCache, block_table, first, cu_tokens, tokens: int,
                  max_tokens: Optional[int] = None, dtype: torch.dtype = torch.bfloat16
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(key, value)`` [tokens, heads, dim] in ``dtype``: row ``cu_tokens[b] + i`` holds the values of
    sequence b's token ``first[b] + i``, for i < ``cu_tokens[b + 1] - cu_tokens[b]``.

    ``tokens`` is ``cu_tokens[-1]``, which the caller knows; rows that no sequence covers are
    undefined.  A token whose page is missing reads as NaN.
    """
    ext = _ext or _native()
    if ext:
        out = ext.kv_read(*cache, block_table, first, cu_tokens, tokens, max_tokens, dtype)
        if out is not None:
            return out
    _not_traced("kv_cache_read")
    seqs = block_table.shape[0] if block_table.dim() else 0
    c, t, dev = _cache_args(cache, block_table, ("first", first, seqs),
                            ("cu_tokens", cu_tokens, seqs + 1))
    if dtype not in _DTYPE:
        raise RuntimeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    key = torch.empty(tokens, c.heads, c.dim, dtype=dtype, device=dev)
    value = torch.empty_like(key)
    with torch.cuda.device(dev):
        _rx.call("rxmet_kv_read", ctypes.byref(c), ctypes.byref(t), first.data_ptr(),
                 cu_tokens.data_ptr(), tokens, tokens if max_tokens is None else max_tokens,
                 key.data_ptr(), value.data_ptr(), _DTYPE[dtype], _rx.stream_of(dev))
    return key, value


def kv_cache_attention(query, cache: KVCache, block_table, lengths, cu_query=None,
                       max_query: Optional[int] = None, max_length: Optional[int] = None,
                       scale: Optional[float] = None, causal: bool = True,
                       window: Optional[int] = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` of each query over its sequence's cached tokens, like query.

    query [queries, q_heads, dim] float16 or bfloat16 (any strides of the first two axes), q_heads a
    multiple of the cache's heads: query head h reads cache head ``h // (q_heads // heads)``.
    Rows ``cu_query[b]..cu_query[b + 1]`` (without ``cu_query``: row b) are the last ones of sequence b's
    ``lengths[b]`` tokens, which the cache holds already.  With ``causal`` a query sees the tokens up to its
    own, with ``window`` only the last ``window`` of them; a query that sees nothing gives 0.
    ``scale`` defaults to ``1 / sqrt(dim)``.  Rows that no sequence covers are undefined.  For inference: query
    gets no gradient.

    ``max_query`` and ``max_length`` (the most queries and tokens of a sequence) size the launch; they
    default to all rows and to the table's width.  Larger values in the device vectors are computed
    as well, more slowly.
    """
    ext = _ext or _native()
    if ext:
        out = ext.kv_attention(query, *cache, block_table, lengths, cu_query, max_query, max_length,
                               scale, causal, window)
        if out is not None:
            return out
    _not_traced("kv_cache_attention")
    seqs = block_table.shape[0] if block_table.dim() else 0
    c, t, dev = _cache_args(cache, block_table, ("lengths", lengths, seqs),
                            ("cu_query", cu_query, seqs + 1))
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"query must be float16 or bfloat16, not {query.dtype}")
    if query.dim() != 3 or query.shape[1] < c.heads or query.shape[1] % c.heads:
        raise RuntimeError(f"query must be [queries, q_heads, {c.dim}] with q_heads a multiple of "
                           f"the cache's {c.heads}, not {tuple(query.shape)}")
    n, hq = query.shape[:2]
    query = _tokens(query, "query", dev, hq, c.dim)
    if cu_query is None:
        if n != seqs:
            raise RuntimeError(f"without cu_query there must be one query for each of the {seqs} "
                               f"sequences, not {n}")
        max_query = 1
    if window is not None and window < 1:
        raise RuntimeError(f"window must be at least 1, not {window}")
    if max_query is None:
        max_query = n
    if max_length is None:
        max_length = t.cols * c.page_size
    window = window or 0
    out = torch.empty(n, hq, c.dim, dtype=query.dtype, device=dev)
    lib = _rx.load()
    size = lib.rxmet_kv_attention_workspace_bytes(ctypes.byref(c), seqs, n, hq, max_query,
                                                  max_length, window)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with torch.cuda.device(dev):
        _rx.call("rxmet_kv_attention", ctypes.byref(c), ctypes.byref(t), lengths.data_ptr(),
                 _rx.ptr(cu_query), n, max_query, max_length, query.data_ptr(), query.stride(0),
                 query.stride(1), hq, 1 / math.sqrt(c.dim) if scale is None else scale,
                 int(causal), window, out.data_ptr(), _DTYPE[query.dtype], _rx.ptr(ws),
                 _rx.stream_of(dev))
    return out
