"""Windowed attention on MI355X: the half of a hybrid layer that runs beside its
Gated DeltaNet recurrence (WindowedHybridLayer.mix,
pseudobrain/transplant.py:989-997, sums the two), over plain tensors for
prefill and training and over a paged key-value cache for serving.

    position p sees key j when j <= p and (j > p - window or j < sinks)
    o_p = sum_j softmax_j(scale q_p . k_j) v_j            over the keys p sees

Tensors follow the operator's layouts: q [B,Tq,Hq,D]; k, v [B,Tk,Hk,D] with Hq a
multiple of Hk (query head h reads key head h // (Hq // Hk)). The queries are
the last Tq positions of their sequence's keys, so Tk > Tq continues a cached
prompt. cu_seqlens (int32 [N+1], B == 1) packs N sequences along T.

  window_attention         forward, and backward through autograd
  paged_decode_attention   the newest token (or a few drafted ones) of each
                           sequence against the cache's pages
  paged_cache_write        new keys and values into the pages

float32, bfloat16 and float16; o comes back in q's dtype, lse (the logarithm of
the softmax sums, by which attention over two sets of keys is merged) in
float32. A query that sees no key gets o = 0 and lse = -inf. Widths D up to 256
are zero-padded to 64, 128 or 256 by window_attention, which leaves every
product as it is; caches hold one of those widths. All of it runs on the GPU
only; a missing library or a CPU tensor raises.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .gated_deltanet import _aligned, _pad_last, _require_device, _width_at_least, grad_needed

ATTENTION_HEAD_DIMS = (64, 128, 256)  # widths the kernels are built for
MAX_DRAFT = 16                        # query tokens a sequence may have in paged_decode_attention
_MAX_TOKEN_STRIDE = 1 << 24           # bytes (pbattn_window_fwd)
_NO_GUARD = contextlib.nullcontext()


def _guard(dev: torch.device):
    """The launch goes to the current device: make it the tensors'."""
    return _NO_GUARD if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"attention takes float32, bfloat16 or float16, not {dtype}")
    return _lib.DTYPE_CODES[dtype]


def _window_args(window, sinks) -> tuple[int, int]:
    """(window, 0 for none; sinks) as the C ABI takes them."""
    if window is not None and int(window) < 1:
        raise ValueError(f"window must be at least 1 (None for no window), got {window}")
    if int(sinks) < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return (0 if window is None else min(int(window), 2**31 - 1)), min(int(sinks), 2**31 - 1)


def _strided(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy, as the kernels read it: a dense last axis, the other
    strides and the address multiples of 16 bytes."""
    size = x.element_size()
    steps = [s for n, s in zip(x.shape[:-1], x.stride()) if n > 1]
    if (x.shape[-1] > 1 and x.stride(-1) != 1) or any(s * size % 16 for s in steps) or (
            x.ndim > 2 and x.stride(-3) * size >= _MAX_TOKEN_STRIDE and x.shape[-3] > 1):
        x = x.contiguous()
    return _aligned(x, 16)


def _strides(*tensors) -> ctypes.Array:
    """Element strides of every axis but the last (0 for axes of one element)."""
    out = [s if n > 1 else 0 for x in tensors for n, s in zip(x.shape[:-1], x.stride())]
    return (ctypes.c_int64 * len(out))(*out)


# ----------------------------------------------------------------------------
# Prefill and training.
# ----------------------------------------------------------------------------
def _window_shapes(q, k, v, cu_q, cu_k):
    """Checked sizes (B, Tq, Tk, Hq, Hk, D) and the number of sequences."""
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape:
        raise ValueError("expected q [B,Tq,Hq,D] and k, v [B,Tk,Hk,D] of one shape")
    batch, tq, hq, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    if k.shape[0] != batch or k.shape[3] != d:
        raise ValueError("k and v must share q's batch axis and head width")
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError("query heads must be a multiple of the key heads")
    if d < 1 or d > ATTENTION_HEAD_DIMS[-1]:
        raise ValueError(f"no attention kernel for head widths above {ATTENTION_HEAD_DIMS[-1]} (got {d})")
    nseq = batch
    if cu_q is None:
        if cu_k is not None:
            raise ValueError("cu_seqlens_k needs cu_seqlens")
    else:
        if batch != 1:
            raise ValueError("cu_seqlens needs B == 1 (sequences packed along T)")
        if cu_q.ndim != 1 or cu_q.numel() < 1:
            raise ValueError("cu_seqlens must be a 1-D tensor [N+1]")
        if cu_k is None and tk != tq:
            raise ValueError("q and k of different lengths need cu_seqlens_k beside cu_seqlens")
        if cu_k is not None and cu_k.shape != cu_q.shape:
            raise ValueError("cu_seqlens_k must have cu_seqlens' shape")
        nseq = cu_q.numel() - 1
    return (batch, tq, tk, hq, hk, d), nseq


def _boundaries(cu):
    return None if cu is None else cu.to(torch.int32).contiguous()


def window_attention_fwd(q, k, v, scale: float, window=None, sinks: int = 0, cu_seqlens=None, cu_seqlens_k=None, *,
                         out: torch.Tensor | None = None, return_lse: bool = True):
    """Launch pbattn_window_fwd at one of the built widths. Returns (o [B,Tq,Hq,D]
    in q's dtype, lse [B,Tq,Hq] float32 or None). k and v are cast to q's dtype;
    `out` may supply o. No backward (window_attention has one)."""
    (batch, tq, tk, hq, hk, d), nseq = _window_shapes(q, k, v, cu_seqlens, cu_seqlens_k)
    dev = _require_device(q, k, v, cu_seqlens, cu_seqlens_k)
    code = _dtype_code(q.dtype)
    if d not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"attention kernels are built for head widths {ATTENTION_HEAD_DIMS}")
    window, sinks = _window_args(window, sinks)
    q, k, v = _strided(q), _strided(k.to(q.dtype)), _strided(v.to(q.dtype))
    cu_q, cu_k = _boundaries(cu_seqlens), _boundaries(cu_seqlens_k)
    if out is None:
        out = torch.empty(batch, tq, hq, d, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of q's shape and dtype")
    if nseq == 0:
        out.zero_()
    lse = torch.empty(batch, tq, hq, dtype=torch.float32, device=dev) if return_lse else None
    if nseq == 0 and return_lse:
        lse.fill_(-torch.inf)
    with _guard(dev):
        status = _lib.attn_lib().pbattn_window_fwd(
            _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), code, _strides(q, k, v), _lib.ptr(cu_q), _lib.ptr(cu_k), nseq,
            _lib.ptr(out), _lib.ptr(lse), batch, tq, tk, hq, hk, d, float(scale), window, sinks,
            _lib.stream_handle(dev))
    _lib.check(status, "pbattn_window_fwd")
    return out, lse


def window_attention_bwd(q, k, v, o, lse, grad_o, scale: float, window=None, sinks: int = 0, cu_seqlens=None,
                         cu_seqlens_k=None, grad_lse=None):
    """Launch pbattn_window_bwd: (dq, dk, dv) in q's dtype from the forward call's
    inputs and results and the gradients of o and (optionally) lse."""
    (batch, tq, tk, hq, hk, d), nseq = _window_shapes(q, k, v, cu_seqlens, cu_seqlens_k)
    dev = _require_device(q, k, v, o, lse, grad_o, grad_lse, cu_seqlens, cu_seqlens_k)
    code = _dtype_code(q.dtype)
    if d not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"attention kernels are built for head widths {ATTENTION_HEAD_DIMS}")
    if o.shape != q.shape or grad_o.shape != q.shape or lse.shape != q.shape[:3] or (
            grad_lse is not None and grad_lse.shape != q.shape[:3]):
        raise ValueError("o and grad_o must have q's shape, lse and grad_lse [B,Tq,Hq]")
    window, sinks = _window_args(window, sinks)
    q, k, v = _strided(q), _strided(k.to(q.dtype)), _strided(v.to(q.dtype))
    o, grad_o = (_aligned(x.to(q.dtype).contiguous(), 16) for x in (o, grad_o))
    lse = lse.to(torch.float32).contiguous()
    grad_lse = None if grad_lse is None else grad_lse.to(torch.float32).contiguous()
    cu_q, cu_k = _boundaries(cu_seqlens), _boundaries(cu_seqlens_k)
    dq = torch.empty(batch, tq, hq, d, dtype=q.dtype, device=dev)
    dk, dv = (torch.empty(batch, tk, hk, d, dtype=q.dtype, device=dev) for _ in range(2))
    if nseq == 0 or tq == 0:
        for x in (dq, dk, dv):
            x.zero_()
        return dq, dk, dv
    with _guard(dev):
        lib = _lib.attn_lib()
        nbytes = lib.pbattn_window_bwd_workspace_size(batch, tq, tk, hq, hk, d, nseq, code, int(cu_q is not None),
                                                      window, sinks)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        status = lib.pbattn_window_bwd(
            _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), code, _strides(q, k, v), _lib.ptr(cu_q), _lib.ptr(cu_k), nseq,
            _lib.ptr(o), _lib.ptr(lse), _lib.ptr(grad_o), _lib.ptr(grad_lse), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv),
            batch, tq, tk, hq, hk, d, float(scale), window, sinks, _lib.ptr(workspace), nbytes,
            _lib.stream_handle(dev))
    _lib.check(status, "pbattn_window_bwd")
    return dq, dk, dv


@torch.library.custom_op("pbgdn::window_attention", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor v, float scale, int? window, int sinks, "
                                "Tensor? cu_seqlens, Tensor? cu_seqlens_k) -> (Tensor, Tensor)")
def window_attention_op(q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    """(o, lse) of window_attention at one of the built widths."""
    return window_attention_fwd(q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k)


@window_attention_op.register_fake
def _(q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


@torch.library.custom_op("pbgdn::window_attention_backward", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor grad_o, "
                                "Tensor? grad_lse, float scale, int? window, int sinks, Tensor? cu_seqlens, "
                                "Tensor? cu_seqlens_k) -> (Tensor, Tensor, Tensor)")
def window_attention_backward_op(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    """(dq, dk, dv) in q's dtype (window_attention_bwd)."""
    return window_attention_bwd(q, k, v, o, lse, grad_o, scale, window, sinks, cu_seqlens, cu_seqlens_k, grad_lse)


@window_attention_backward_op.register_fake
def _(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    return q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(v.shape)


def _attention_setup(ctx, inputs, output):
    q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k = inputs
    o, lse = output
    ctx.save_for_backward(q, k, v, o, lse, cu_seqlens, cu_seqlens_k)
    ctx.scale, ctx.window, ctx.sinks = scale, window, sinks
    ctx.set_materialize_grads(False)


def _attention_grad(ctx, grad_o, grad_lse):
    if grad_o is None and grad_lse is None:
        return (None,) * 8
    q, k, v, o, lse, cu_seqlens, cu_seqlens_k = ctx.saved_tensors
    grad_o = torch.zeros_like(o) if grad_o is None else grad_o
    dq, dk, dv = window_attention_backward_op(q, k, v, o, lse, grad_o, grad_lse, ctx.scale, ctx.window, ctx.sinks,
                                              cu_seqlens, cu_seqlens_k)
    return dq, dk.to(k.dtype), dv.to(v.dtype), None, None, None, None, None


window_attention_op.register_autograd(_attention_grad, setup_context=_attention_setup)


def window_attention(q, k, v, scale: float, window=None, sinks: int = 0, cu_seqlens=None, cu_seqlens_k=None, *,
                     return_lse: bool = False):
    """Attention with a sliding window of `window` keys (the query's own among
    them; None for every earlier key) and the first `sinks` keys of the sequence
    always visible. q [B,Tq,Hq,D], k, v [B,Tk,Hk,D], the queries at the sequence's
    last Tq positions; cu_seqlens (and cu_seqlens_k, where keys and queries differ
    in number) packs sequences. Returns o [B,Tq,Hq,D] in q's dtype, with
    return_lse (o, lse [B,Tq,Hq] float32); differentiable in q, k and v, also
    through lse."""
    shapes, _ = _window_shapes(q, k, v, cu_seqlens, cu_seqlens_k)
    _require_device(q, k, v, cu_seqlens, cu_seqlens_k)
    _dtype_code(q.dtype)
    _window_args(window, sinks)
    d = shapes[-1]
    width = _width_at_least(d, ATTENTION_HEAD_DIMS)
    if width != d:
        q, k, v = (_pad_last(x, width) for x in (q, k, v))
    if grad_needed(q, k, v) or torch.compiler.is_compiling():
        window = None if window is None else int(window)
        o, lse = window_attention_op(q, k, v, float(scale), window, int(sinks), cu_seqlens, cu_seqlens_k)
    else:
        o, lse = window_attention_fwd(q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k, return_lse=return_lse)
    if width != d:
        o = o[..., :d].contiguous()
    return (o, lse) if return_lse else o


# ----------------------------------------------------------------------------
# The paged cache.
# ----------------------------------------------------------------------------
def _inference_only(where: str, *tensors) -> None:
    if grad_needed(*tensors):
        raise RuntimeError(f"{where} has no backward: call it under torch.no_grad() (inference), or use "
                           "window_attention, which has one")


def _caches(k_cache, v_cache):
    """Checked caches [pages, page, Hk, D] of equal strides (any axis order with
    the token rows of a page evenly spaced): (pages, page, Hk, D) and the strides."""
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("expected k_cache and v_cache [pages, page, Hk, D] of one shape and dtype")
    pages, page, hk, d = k_cache.shape
    if page < 1 or hk < 1:
        raise ValueError("a cache has at least one token a page and one head")
    size = k_cache.element_size()
    strides = k_cache.stride()
    if (strides != v_cache.stride() or strides[3] != 1 or any(s * size % 16 for s in strides[:3])
            or strides[1] < 1 or strides[0] % strides[1] or k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16):
        raise ValueError("caches must have equal strides, a dense last axis, page strides that are multiples of the "
                         "token stride, and strides and addresses that are multiples of 16 bytes")
    return (pages, page, hk, d), (ctypes.c_int64 * 3)(*strides[:3])


def _decode(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out=None, return_lse=False):
    if q.ndim != 4:
        raise ValueError("expected q [B,T,Hq,D]")
    batch, length, hq, d = q.shape
    dev = _require_device(q, k_cache, v_cache, page_table, lengths)
    (pages, page, hk, dc), strides = _caches(k_cache, v_cache)
    code = _dtype_code(k_cache.dtype)
    if q.dtype != k_cache.dtype:
        raise ValueError(f"q ({q.dtype}) and the caches ({k_cache.dtype}) must have one dtype")
    if d != dc or hq < 1 or hq % hk:
        raise ValueError("q must have the caches' head width and a multiple of their heads")
    if d not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"cached heads must have a width in {ATTENTION_HEAD_DIMS}")
    if not 1 <= length <= MAX_DRAFT:
        raise ValueError(f"paged decoding takes 1 to {MAX_DRAFT} query tokens a sequence, got {length}")
    if page_table.ndim != 2 or page_table.shape[0] != batch or lengths.shape != (batch,):
        raise ValueError("expected page_table [B, max_pages] and lengths [B]")
    window, sinks = _window_args(window, sinks)
    q = _aligned(q.contiguous(), 16)
    if page_table.dtype != torch.int32 or not page_table.is_contiguous():
        page_table = page_table.to(torch.int32).contiguous()
    if lengths.dtype != torch.int32 or not lengths.is_contiguous():
        lengths = lengths.to(torch.int32).contiguous()
    if out is None:
        out = torch.empty(batch, length, hq, d, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of q's shape and dtype")
    lse = torch.empty(batch, length, hq, dtype=torch.float32, device=dev) if return_lse else None
    with _guard(dev):
        lib = _lib.attn_lib()
        nbytes = lib.pbattn_paged_decode_workspace_size(batch, length, hq, hk, d)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        status = lib.pbattn_paged_decode(
            _lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(v_cache), code, strides, page, pages, _lib.ptr(page_table),
            page_table.shape[1], _lib.ptr(lengths), _lib.ptr(out), _lib.ptr(lse), batch, length, hq, hk, d,
            float(scale), window, sinks, _lib.ptr(workspace), nbytes, _lib.stream_handle(dev))
    _lib.check(status, "pbattn_paged_decode")
    return out, lse


@torch.library.custom_op("pbgdn::paged_decode_attention", mutates_args=(),
                         schema="(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor lengths, "
                                "float scale, int? window, int sinks) -> (Tensor, Tensor)")
def paged_decode_attention_op(q, k_cache, v_cache, page_table, lengths, scale, window, sinks):
    """(o, lse) of paged_decode_attention."""
    return _decode(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, return_lse=True)


@paged_decode_attention_op.register_fake
def _(q, k_cache, v_cache, page_table, lengths, scale, window, sinks):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


def paged_decode_attention(q, k_cache, v_cache, page_table, lengths, scale: float, window=None, sinks: int = 0, *,
                           return_lse: bool = False, out: torch.Tensor | None = None):
    """One decode step: q [B,T,Hq,D], the T newest tokens of each sequence (1, or
    the sampled token and drafted ones), against keys and values in pages.
    k_cache, v_cache [pages, page, Hk, D] (any strides with dense rows evenly
    spaced in a page); page_table [B, max_pages] int32: key j of sequence b lies
    in page page_table[b, j // page]; lengths [B] int32: the sequence's cached
    keys, those of the T tokens among them, so that token t stands at position
    lengths[b] - T + t. Pages that no token sees need no entry (a sliding window
    frees them); the keys of an entry outside the cache count as absent, and a
    sequence of length 0 (padding) gives zeros. window and sinks as in
    window_attention. Returns o [B,T,Hq,D] in q's dtype, with return_lse (o, lse
    [B,T,Hq] float32). Inference only."""
    _inference_only("paged_decode_attention", q, k_cache, v_cache)
    if torch.compiler.is_compiling() and out is None:
        o, lse = paged_decode_attention_op(q, k_cache, v_cache, page_table, lengths, float(scale), window, int(sinks))
    else:
        o, lse = _decode(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out, return_lse)
    return (o, lse) if return_lse else o


def _write(k, v, k_cache, v_cache, slots):
    dev = _require_device(k, v, k_cache, v_cache, slots)
    (pages, page, hk, d), strides = _caches(k_cache, v_cache)
    code = _dtype_code(k_cache.dtype)
    if k.ndim < 3 or v.shape != k.shape or k.shape[-2:] != (hk, d) or slots.shape != k.shape[:-2]:
        raise ValueError("expected k, v [..., Hk, D] with the caches' heads and slots [...]")
    if slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slots must be int32 or int64")
    k, v = (_strided(x.to(k_cache.dtype).reshape(-1, hk, d)) for x in (k, v))
    slots = slots.reshape(-1).to(torch.int64).contiguous()
    with _guard(dev):
        status = _lib.attn_lib().pbattn_paged_write(
            _lib.ptr(k), _lib.ptr(v), code, _strides(k, v), _lib.ptr(k_cache), _lib.ptr(v_cache), strides, page, pages,
            _lib.ptr(slots), slots.numel(), hk, d, _lib.stream_handle(dev))
    _lib.check(status, "pbattn_paged_write")


@torch.library.custom_op("pbgdn::paged_cache_write_", mutates_args=("k_cache", "v_cache"),
                         schema="(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots) -> ()")
def paged_cache_write_op(k, v, k_cache, v_cache, slots):
    """paged_cache_write, for graphs of ops."""
    _write(k, v, k_cache, v_cache, slots)


@paged_cache_write_op.register_fake
def _(k, v, k_cache, v_cache, slots):
    return None


def paged_cache_write(k, v, k_cache, v_cache, slots) -> None:
    """Write keys and values k, v [..., Hk, D] into the pages of k_cache and v_cache
    [pages, page, Hk, D] in place: the token at slots[...] = s goes to row s % page
    of page s // page. A slot outside the cache (e.g. -1 for padding) is skipped;
    the others must be distinct. k and v are cast to the caches' dtype. Inference
    only."""
    _inference_only("paged_cache_write", k, v, k_cache, v_cache)
    if torch.compiler.is_compiling():
        paged_cache_write_op(k, v, k_cache, v_cache, slots)
    else:
        _write(k, v, k_cache, v_cache, slots)
