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

import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .gated_deltanet import _aligned, _pad_last, _require_device, _width_at_least, grad_needed

ATTENTION_HEAD_DIMS = (64, 128, 256)  # widths the kernels are built for
MAX_DRAFT = 16                        # query tokens a sequence may have in paged_decode_attention
_MAX_TOKEN_STRIDE = 1 << 24           # bytes (pbattn_window_fwd)
_MAX_TILE_SPAN = 0x7ffffff0           # bytes (pbattn_window_bwd)


# What follows from shapes, strides and types alone (checks, stride arrays,
# workspace sizes) is kept by them: a decode step's calls repeat them, and are
# short enough that working it out again would be most of their time.
_plan = functools.lru_cache(maxsize=1024)


def _launch(where: str, fn, dev: torch.device, *args) -> None:
    """fn(*args, stream) on the tensors' device, which need not be the current one."""
    if torch.cuda.current_device() == dev.index:
        status = fn(*args, _lib.stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _lib.stream_handle(dev))
    if status:
        _lib.check(status, where)


def _one_device(first, *rest) -> torch.device:
    """The tensors' device, by _require_device's rules and errors."""
    index = first.get_device()
    if index < 0:
        return _require_device(first, *rest)
    for t in rest:
        if t is not None and t.get_device() != index:
            return _require_device(first, *rest)
    return first.device


def _no_tangents(where: str, *tensors) -> None:
    """Raise where forward-mode differentiation would lose the tensors' tangents."""
    if forward_ad._current_level >= 0 and not _compiling() and any(
            [t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors]):
        raise RuntimeError(f"{where} has no forward-mode derivative")


# (bound once: a short call asks all of them)
_compiling, _dispatch_modes = torch.compiler.is_compiling, torch._C._len_torch_dispatch_stack
_transformed, _tracing = torch._C._are_functorch_transforms_active, torch._C._get_tracing_state
_increment_version = torch.autograd.graph.increment_version
_plain = frozenset((torch.Tensor, torch.nn.Parameter)).issuperset


def _untraced(*tensors) -> bool:
    """Ordinary tensors that nothing compiles, traces or transforms."""
    return not (_compiling() or _dispatch_modes() or _transformed() or _tracing()) and _plain(map(type, tensors))


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"attention takes float32, bfloat16 or float16, not {dtype}")
    return _lib.DTYPE_CODES[dtype]


def _window_args(window, sinks) -> tuple[int, int]:
    """(window, 0 for none; sinks) as the C ABI takes them."""
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 (None for no window), got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return (0 if window is None else min(window, 2**31 - 1)), min(sinks, 2**31 - 1)


def _readable(shape, stride, size: int) -> bool:
    """The kernels read a tensor of these strides in place: a dense last axis, the
    other strides multiples of 16 bytes, token rows less than 16 MiB apart."""
    if shape[-1] > 1 and stride[-1] != 1:
        return False
    if len(shape) > 2 and shape[-3] > 1 and stride[-3] * size >= _MAX_TOKEN_STRIDE:
        return False
    return all(n <= 1 or st * size % 16 == 0 for n, st in zip(shape[:-1], stride))


def _steps(*views) -> ctypes.Array:
    """Element strides of every axis but the last (0 for axes of one element)."""
    out = [st if n > 1 else 0 for shape, stride in views for n, st in zip(shape[:-1], stride)]
    return (ctypes.c_int64 * len(out))(*out)


# ----------------------------------------------------------------------------
# Prefill and training.
# ----------------------------------------------------------------------------
@_plan
def _window_plan(q, k, v, dtype, cu_q, cu_k, window, sinks):
    """Checked sizes (B, Tq, Tk, Hq, Hk, D) and number of sequences of a call with
    q, k, v, boundaries of these shapes, its dtype code, window and sinks."""
    if len(q) != 4 or len(k) != 4 or v != k:
        raise ValueError("expected q [B,Tq,Hq,D] and k, v [B,Tk,Hk,D] of one shape")
    batch, tq, hq, d = q
    tk, hk = k[1], k[2]
    if k[0] != batch or k[3] != d:
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
        if len(cu_q) != 1 or cu_q[0] < 1:
            raise ValueError("cu_seqlens must be a 1-D tensor [N+1]")
        if cu_k is None and tk != tq:
            raise ValueError("q and k of different lengths need cu_seqlens_k beside cu_seqlens")
        if cu_k is not None and cu_k != cu_q:
            raise ValueError("cu_seqlens_k must have cu_seqlens' shape")
        nseq = cu_q[0] - 1
    return ((batch, tq, tk, hq, hk, d), nseq, _dtype_code(dtype), *_window_args(window, sinks))


def _shape(x):
    return None if x is None else x.shape


def _window_check(q, k, v, cu_q, cu_k, window, sinks):
    return _window_plan(q.shape, k.shape, v.shape, q.dtype, _shape(cu_q), _shape(cu_k),
                        None if window is None else int(window), int(sinks))


@_plan
def _window_steps(q, k, v, size):
    """The stride array of q, k, v by their (shape, stride), None if one is not readable in place."""
    return _steps(q, k, v) if all(_readable(*x, size) for x in (q, k, v)) else None


@_plan
def _tile_span(q, stride, hk: int, size: int) -> int:
    """Bytes from the first to the last element of a gradient kernel's tile of q: 32
    rows, the heads of a group (32 at most) of as many tokens as there is room for."""
    heads = min(q[2] // hk, 32)
    steps = (32 // heads - 1, stride[1] if q[1] > 1 else 0), (heads - 1, stride[2] if q[2] > 1 else 0), (q[3], 1)
    return sum(n * step for n, step in steps) * size


def _window_operands(q, k, v, gradients: bool = False):
    """q, k, v in q's dtype as the kernels (those of the gradients too) read them, and
    their stride array."""
    if k.dtype != q.dtype or v.dtype != q.dtype:
        k, v = k.to(q.dtype), v.to(q.dtype)
    # (the strides are taken last: a copy for the alignment may have others than its view)
    q, k, v = _aligned(q, 16), _aligned(k, 16), _aligned(v, 16)
    if gradients and _tile_span(q.shape, q.stride(), k.shape[2], q.element_size()) > _MAX_TILE_SPAN:
        q = q.contiguous()
    steps = _window_steps((q.shape, q.stride()), (k.shape, k.stride()), (v.shape, v.stride()), q.element_size())
    if steps is None:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        steps = _steps(*((x.shape, x.stride()) for x in (q, k, v)))
    return q, k, v, steps


def _boundaries(cu):
    if cu is None or (cu.dtype == torch.int32 and cu.is_contiguous()):
        return cu
    return cu.to(torch.int32).contiguous()


def _output(out, q):
    """The output tensor of a call with these q: `out`, or a new dense one."""
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of q's shape and dtype")
    return out


def _built_width(d: int) -> None:
    if d not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"attention kernels are built for head widths {ATTENTION_HEAD_DIMS}")


def window_attention_fwd(q, k, v, scale: float, window=None, sinks: int = 0, cu_seqlens=None, cu_seqlens_k=None, *,
                         out: torch.Tensor | None = None, return_lse: bool = True):
    """Launch pbattn_window_fwd at one of the built widths. Returns (o [B,Tq,Hq,D]
    in q's dtype, lse [B,Tq,Hq] float32 or None). k and v are cast to q's dtype;
    `out` may supply o. No backward (window_attention has one)."""
    sizes, nseq, code, window, sinks = _window_check(q, k, v, cu_seqlens, cu_seqlens_k, window, sinks)
    dev = _one_device(q, k, v, cu_seqlens, cu_seqlens_k)
    _built_width(sizes[-1])
    q, k, v, steps = _window_operands(q, k, v)
    cu_q, cu_k = _boundaries(cu_seqlens), _boundaries(cu_seqlens_k)
    out = _output(out, q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if return_lse else None
    if nseq == 0:
        out.zero_()
        if return_lse:
            lse.fill_(-torch.inf)
    _launch("pbattn_window_fwd", _lib.attn_lib().pbattn_window_fwd, dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), code,
            steps, _lib.ptr(cu_q), _lib.ptr(cu_k), nseq, out.data_ptr(), _lib.ptr(lse), *sizes, float(scale), window, sinks)
    return out, lse


def window_attention_bwd(q, k, v, o, lse, grad_o, scale: float, window=None, sinks: int = 0, cu_seqlens=None,
                         cu_seqlens_k=None, grad_lse=None):
    """Launch pbattn_window_bwd: (dq, dk, dv) in q's dtype from the forward call's
    inputs and results and the gradients of o and (optionally) lse."""
    sizes, nseq, code, window, sinks = _window_check(q, k, v, cu_seqlens, cu_seqlens_k, window, sinks)
    dev = _one_device(q, k, v, o, lse, grad_o, grad_lse, cu_seqlens, cu_seqlens_k)
    _built_width(sizes[-1])
    if o.shape != q.shape or grad_o.shape != q.shape or lse.shape != q.shape[:3] or (
            grad_lse is not None and grad_lse.shape != q.shape[:3]):
        raise ValueError("o and grad_o must have q's shape, lse and grad_lse [B,Tq,Hq]")
    q, k, v, steps = _window_operands(q, k, v, gradients=True)
    o, grad_o = (_aligned(x.to(q.dtype).contiguous(), 16) for x in (o, grad_o))
    lse = lse.to(torch.float32).contiguous()
    grad_lse = None if grad_lse is None else grad_lse.to(torch.float32).contiguous()
    cu_q, cu_k = _boundaries(cu_seqlens), _boundaries(cu_seqlens_k)
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
    dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=dev) for _ in range(2))
    if nseq == 0 or sizes[1] == 0:
        for x in (dq, dk, dv):
            x.zero_()
        return dq, dk, dv
    lib = _lib.attn_lib()
    with torch.cuda.device(dev):  # (the size depends on the device's compute units)
        nbytes = lib.pbattn_window_bwd_workspace_size(*sizes, nseq, code, int(cu_q is not None), window, sinks)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch("pbattn_window_bwd", lib.pbattn_window_bwd, dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), code, steps,
            _lib.ptr(cu_q), _lib.ptr(cu_k), nseq, o.data_ptr(), lse.data_ptr(), grad_o.data_ptr(), _lib.ptr(grad_lse),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *sizes, float(scale), window, sinks, workspace.data_ptr(), nbytes)
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


def _backward_launch(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    return window_attention_bwd(q, k, v, o, lse, grad_o, scale, window, sinks, cu_seqlens, cu_seqlens_k, grad_lse)


@torch.library.custom_op("pbgdn::window_attention_backward", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor grad_o, "
                                "Tensor? grad_lse, float scale, int? window, int sinks, Tensor? cu_seqlens, "
                                "Tensor? cu_seqlens_k) -> (Tensor, Tensor, Tensor)")
def window_attention_backward_op(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    """(dq, dk, dv) in q's dtype (window_attention_bwd)."""
    return _backward_launch(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k)


@window_attention_backward_op.register_fake
def _(q, k, v, o, lse, grad_o, grad_lse, scale, window, sinks, cu_seqlens, cu_seqlens_k):
    return q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(v.shape)


def _attention_setup(ctx, inputs, output):
    q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k = inputs
    o, lse = output
    ctx.save_for_backward(q, k, v, o, lse, cu_seqlens, cu_seqlens_k)
    ctx.scale, ctx.window, ctx.sinks = scale, window, sinks
    ctx.set_materialize_grads(False)


def _gradients(backward):
    """The backward formula, by `backward`: the op, or its launch itself."""
    def formula(ctx, grad_o, grad_lse):
        if grad_o is None and grad_lse is None:
            return (None,) * 8
        q, k, v, o, lse, cu_seqlens, cu_seqlens_k = ctx.saved_tensors
        grad_o = torch.zeros_like(o) if grad_o is None else grad_o
        dq, dk, dv = backward(q, k, v, o, lse, grad_o, grad_lse, ctx.scale, ctx.window, ctx.sinks, cu_seqlens,
                              cu_seqlens_k)
        return dq, dk.to(k.dtype), dv.to(v.dtype), None, None, None, None, None
    return formula


window_attention_op.register_autograd(_gradients(window_attention_backward_op), setup_context=_attention_setup)


class _WindowAttention(torch.autograd.Function):
    """The op and its gradients without the op's dispatch, which costs more than a short call."""
    _launched = staticmethod(_gradients(_backward_launch))
    _traced = staticmethod(_gradients(window_attention_backward_op))

    @staticmethod
    def forward(ctx, *inputs):
        output = window_attention_fwd(*inputs)
        _attention_setup(ctx, inputs, output)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_o, grad_lse):
        _no_tangents("window_attention's backward", grad_o, grad_lse)
        tensors = [t for t in (grad_o, grad_lse) if t is not None]
        return (_WindowAttention._launched if _untraced(*tensors) else _WindowAttention._traced)(ctx, grad_o, grad_lse)


def window_attention(q, k, v, scale: float, window=None, sinks: int = 0, cu_seqlens=None, cu_seqlens_k=None, *,
                     return_lse: bool = False):
    """Attention with a sliding window of `window` keys (the query's own among
    them; None for every earlier key) and the first `sinks` keys of the sequence
    always visible. q [B,Tq,Hq,D], k, v [B,Tk,Hk,D], the queries at the sequence's
    last Tq positions; cu_seqlens (and cu_seqlens_k, where keys and queries differ
    in number) packs sequences. Returns o [B,Tq,Hq,D] in q's dtype, with
    return_lse (o, lse [B,Tq,Hq] float32); differentiable in q, k and v, also
    through lse, once and in reverse mode (a forward-mode tangent raises)."""
    _no_tangents("window_attention", q, k, v)
    d = _window_check(q, k, v, cu_seqlens, cu_seqlens_k, window, sinks)[0][-1]
    _one_device(q, k, v, cu_seqlens, cu_seqlens_k)
    if d not in ATTENTION_HEAD_DIMS:
        q, k, v = (_pad_last(x, _width_at_least(d, ATTENTION_HEAD_DIMS)) for x in (q, k, v))
    traced = not _untraced(q, k, v)
    if traced or grad_needed(q, k, v):
        window = None if window is None else int(window)
        o, lse = (window_attention_op if traced else _WindowAttention.apply)(q, k, v, float(scale), window, int(sinks), cu_seqlens, cu_seqlens_k)
    else:
        o, lse = window_attention_fwd(q, k, v, scale, window, sinks, cu_seqlens, cu_seqlens_k, return_lse=return_lse)
    if d not in ATTENTION_HEAD_DIMS:
        o = o[..., :d].contiguous()
    return (o, lse) if return_lse else o


# ----------------------------------------------------------------------------
# The paged cache.
# ----------------------------------------------------------------------------
def _inference_only(where: str, *tensors) -> None:
    if forward_ad._current_level >= 0:
        _no_tangents(where, *tensors)
    if torch.is_grad_enabled() and any([t.requires_grad for t in tensors]):
        raise RuntimeError(f"{where} has no backward: call it under torch.no_grad() (inference), or use "
                           "window_attention, which has one")


@_plan
def _cache_plan(shape, stride, v_shape, v_stride, dtype, v_dtype):
    """Checked sizes (pages, page, Hk, D) of caches of these shapes and strides, the
    stride array and the dtype code."""
    if len(shape) != 4 or v_shape != shape or v_dtype != dtype:
        raise ValueError("expected k_cache and v_cache [pages, page, Hk, D] of one shape and dtype")
    if shape[1] < 1 or shape[2] < 1:
        raise ValueError("a cache has at least one token a page and one head")
    code = _dtype_code(dtype)
    if (stride != v_stride or stride[3] != 1 or any(s * dtype.itemsize % 16 for s in stride[:3]) or stride[1] < 1
            or stride[0] % stride[1]):
        raise ValueError("caches must have equal strides, a dense last axis, page strides that are multiples of the "
                         "token stride, and strides that are multiples of 16 bytes")
    return tuple(shape), (ctypes.c_int64 * 3)(*stride[:3]), code


def _caches(k_cache, v_cache):
    """_cache_plan of two caches, and their addresses."""
    plan = _cache_plan(k_cache.shape, k_cache.stride(), v_cache.shape, v_cache.stride(), k_cache.dtype, v_cache.dtype)
    at = k_cache.data_ptr(), v_cache.data_ptr()
    if (at[0] | at[1]) % 16:
        raise ValueError("caches must be aligned to 16 bytes")
    return (*plan, at)


@_plan
def _decode_plan(q, q_dtype, cache, table, lengths, window, sinks, device_index: int):
    """What a decode call with tensors of these shapes passes on: its checked sizes
    (B, T, Hq, Hk, D), window, sinks, and the workspace's bytes on the device."""
    (_, _, hk, dc), dtype = cache
    if q_dtype != dtype:
        raise ValueError(f"q ({q_dtype}) and the caches ({dtype}) must have one dtype")
    if len(q) != 4:
        raise ValueError("expected q [B,T,Hq,D]")
    batch, length, hq, d = q
    if d != dc or hq < 1 or hq % hk:
        raise ValueError("q must have the caches' head width and a multiple of their heads")
    if d not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"cached heads must have a width in {ATTENTION_HEAD_DIMS}")
    if not 1 <= length <= MAX_DRAFT:
        raise ValueError(f"paged decoding takes 1 to {MAX_DRAFT} query tokens a sequence, got {length}")
    if len(table) != 2 or table[0] != batch or lengths != (batch,):
        raise ValueError("expected page_table [B, max_pages] and lengths [B]")
    sizes = (batch, length, hq, hk, d)
    with torch.cuda.device(device_index):  # (the workspace depends on the device's compute units)
        nbytes = _lib.attn_lib().pbattn_paged_decode_workspace_size(*sizes)
    return sizes, *_window_args(window, sinks), nbytes


def _decode(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out=None, return_lse=False):
    dev = _one_device(q, k_cache, v_cache, page_table, lengths)
    cache, steps, code, at = _caches(k_cache, v_cache)
    sizes, window, sinks, nbytes = _decode_plan(
        q.shape, q.dtype, (cache, k_cache.dtype), page_table.shape, lengths.shape,
        None if window is None else int(window), int(sinks), dev.index)
    q = _aligned(q.contiguous(), 16)
    page_table, lengths = _boundaries(page_table), _boundaries(lengths)
    out = _output(out, q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if return_lse else None
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch("pbattn_paged_decode", _lib.attn_lib().pbattn_paged_decode, dev, q.data_ptr(), *at, code, steps, cache[1],
            cache[0], page_table.data_ptr(), page_table.shape[1], lengths.data_ptr(), out.data_ptr(), _lib.ptr(lse),
            *sizes, float(scale), window, sinks, workspace.data_ptr(), nbytes)
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
    if _untraced(q, k_cache, v_cache, page_table, lengths):
        o, lse = _decode(q, k_cache, v_cache, page_table, lengths, scale, window, sinks, out, return_lse)
    else:
        window = None if window is None else int(window)
        o, lse = paged_decode_attention_op(q, k_cache, v_cache, page_table, lengths, float(scale), window, int(sinks))
        if out is not None:
            if out.shape != o.shape or out.dtype != o.dtype:
                raise ValueError("out must have q's shape and dtype")
            o = out.copy_(o)
    return (o, lse) if return_lse else o


@_plan
def _write_steps(cache, k, k_stride, v, v_stride, slots, size):
    """The stride array of new rows of these shapes, None if they are not readable
    as [N, Hk, D] in place."""
    if len(k) < 3 or v != k or k[-2:] != cache[2:] or slots != k[:-2]:
        raise ValueError("expected k, v [..., Hk, D] with the caches' heads and slots [...]")
    if len(k) != 3 or not (_readable(k, k_stride, size) and _readable(v, v_stride, size)):
        return None
    return _steps((k, k_stride), (v, v_stride))


def _write_operands(k, v, cache, dtype, slots_shape):
    """New rows in the caches' dtype as the kernel reads them, and their stride array."""
    if (k.data_ptr() | v.data_ptr()) % 16:  # (before the strides are taken: a copy may have others)
        k, v = _aligned(k, 16), _aligned(v, 16)
    steps = _write_steps(cache, k.shape, k.stride(), v.shape, v.stride(), slots_shape, dtype.itemsize)
    if steps is None or k.dtype != dtype or v.dtype != dtype:
        k, v = (x.to(dtype).reshape(-1, *cache[2:]).contiguous() for x in (k, v))
        steps = _steps((k.shape, k.stride()), (v.shape, v.stride()))
    return k, v, steps


def _write(k, v, k_cache, v_cache, slots):
    dev = _one_device(k, v, k_cache, v_cache, slots)
    cache, cache_steps, code, at = _caches(k_cache, v_cache)
    if slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slots must be int32 or int64")
    k, v, steps = _write_operands(k, v, cache, k_cache.dtype, slots.shape)
    if slots.dtype != torch.int64 or slots.ndim != 1 or not slots.is_contiguous():
        slots = slots.reshape(-1).to(torch.int64).contiguous()
    _launch("pbattn_paged_write", _lib.attn_lib().pbattn_paged_write, dev, k.data_ptr(), v.data_ptr(), code, steps, *at,
            cache_steps, cache[1], cache[0], slots.data_ptr(), slots.shape[0], cache[2], cache[3])


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
    if _untraced(k, v, k_cache, v_cache, slots):
        _write(k, v, k_cache, v_cache, slots)
        _increment_version((k_cache, v_cache))  # (as the op does)
    else:
        paged_cache_write_op(k, v, k_cache, v_cache, slots)
