"""The paged key-value cache held in 4 bits, on MI355X: what pseudobrain_amd.attention's
paged operators do, over a cache of a quarter of the size.

32 consecutive values of a head share a scale, a power of two; each is held as the
nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} of it (ties to the even code), the scale
such that the largest of the 32 is 4 or 6 of them: no value is off by more than half
of its step, an eighth to a quarter of its own size (include/pbattn.h says it bit by
bit). 32 values among which one is infinite or NaN read as NaN.

A cache is four uint8 tensors (k, v, k_scale, v_scale): codes [pages, page, Hk, D / 2]
(byte i of a row: value 2 i in the lower half, 2 i + 1 in the upper one) and scales
[pages, page, Hk, D / 32], laid out alike (every stride of the scales a sixteenth of the
codes'). fp4_cache makes one; D is 64, 128 or 256.

  paged_cache_write_fp4        new keys and values into the pages
  paged_decode_attention_fp4   the newest token (or a few drafted ones) of each
                               sequence against the cache's pages
  paged_cache_read_fp4         whole contexts back as rows, for the attention of a
                               prompt's next piece (window_attention)

Inference only, and on the GPU only; a missing library or a CPU tensor raises.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .attention import (
    ATTENTION_HEAD_DIMS, MAX_DRAFT, _boundaries, _dtype_code, _increment_version, _inference_only, _launch, _one_device,
    _output, _plan, _untraced, _window_args, _write_operands,
)
from .gated_deltanet import _aligned

FP4_BLOCK = 32       # values that share a scale
MAX_REQUESTS = 4096  # sequences paged_cache_read_fp4 takes (PBATTN_MAX_REQUESTS)


class Fp4Cache(NamedTuple):
    """Codes and scales of cached keys and values."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def fp4_cache(pages: int, page: int, heads: int, width: int, device="cuda", heads_first: bool = True) -> Fp4Cache:
    """An empty cache of `pages` pages of `page` tokens (zeros: every value 0). heads_first
    lays a page's tokens of one head together, whose rows of D / 2 bytes are then read in
    longer runs; the tensors' axes are [pages, page, heads, ...] either way."""
    if width not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"cached heads must have a width in {ATTENTION_HEAD_DIMS}")
    if pages < 0 or page < 1 or heads < 1:
        raise ValueError("a cache has at least one token a page and one head")
    shape = (pages, heads, page) if heads_first else (pages, page, heads)
    out = [torch.zeros(*shape, n, dtype=torch.uint8, device=device) for n in (width // 2, width // FP4_BLOCK) for _ in "kv"]
    return Fp4Cache(*(x.transpose(1, 2) for x in out)) if heads_first else Fp4Cache(*out)


@_plan
def _fp4_plan(k, k_stride, ks, ks_stride):
    """Checked sizes (pages, page, Hk, D) of a cache of codes and scales of these shapes and
    strides, and the stride array."""
    if len(k) != 4 or len(ks) != 4 or ks[:3] != k[:3] or ks[3] * 16 != k[3]:
        raise ValueError(_FP4_SHAPES)
    pages, page, heads, row = k
    if page < 1 or heads < 1:
        raise ValueError("a cache has at least one token a page and one head")
    if 2 * row not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"cached heads must have a width in {ATTENTION_HEAD_DIMS}")

    def steps(shape, stride):
        """Page, token and head strides in rows, as those of axes of one element follow from the others."""
        if stride[3] != 1 or any(n > 1 and (st < shape[3] or st % shape[3]) for n, st in zip(shape[:3], stride)):
            return None
        p, t, h = (st // shape[3] if n > 1 else 0 for n, st in zip(shape[:3], stride))
        t = t or p or 1
        return p or t * page, t, h

    at = steps(k, k_stride)
    if at is None or at[0] % at[1] or steps(ks, ks_stride) != at:
        raise ValueError(_FP4_LAYOUT)
    return (pages, page, heads, 2 * row), (ctypes.c_int64 * 3)(*(row * x for x in at))


_FP4_SHAPES = "expected a cache of codes k, v [pages, page, Hk, D / 2] and scales [pages, page, Hk, D / 32]"
_FP4_LAYOUT = ("codes and scales must be laid out alike: dense rows, equal strides in rows that are multiples of one (the "
               "scales' a sixteenth of the codes'), pages a whole number of tokens apart")


def _fp4(cache):
    """_fp4_plan of a cache, and its tensors' addresses."""
    k, v, ks, vs = cache
    if not k.dtype == v.dtype == ks.dtype == vs.dtype == torch.uint8:
        raise ValueError("codes and scales are uint8")
    shape, stride, s_shape, s_stride = k.shape, k.stride(), ks.shape, ks.stride()
    if v.shape != shape or vs.shape != s_shape:
        raise ValueError(_FP4_SHAPES)
    plan = _fp4_plan(shape, stride, s_shape, s_stride)
    if (v.stride() != stride or vs.stride() != s_stride) and (
            list(_fp4_plan(shape, v.stride(), s_shape, vs.stride())[1]) != list(plan[1])):
        raise ValueError(_FP4_LAYOUT)
    at = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if (at[0] | at[1] | at[2] | at[3]) % 16:
        raise ValueError("codes and scales must be aligned to 16 bytes")
    return (*plan, at)


# ----------------------------------------------------------------------------
# Decoding.
# ----------------------------------------------------------------------------
@_plan
def _decode_plan(q, dtype, cache, table, lengths, window, sinks, device_index: int):
    """What a decode call with tensors of these shapes passes on: its checked sizes
    (B, T, Hq, Hk, D), q's dtype code, window, sinks, and the workspace's bytes on the device."""
    _, _, hk, dc = cache
    if len(q) != 4:
        raise ValueError("expected q [B,T,Hq,D]")
    batch, length, hq, d = q
    if d != dc or hq < 1 or hq % hk:
        raise ValueError("q must have the cache's head width and a multiple of its heads")
    if not 1 <= length <= MAX_DRAFT:
        raise ValueError(f"paged decoding takes 1 to {MAX_DRAFT} query tokens a sequence, got {length}")
    if len(table) != 2 or table[0] != batch or lengths != (batch,) or table[1] >= 2**31:
        raise ValueError("expected page_table [B, max_pages] and lengths [B]")
    code, sizes = _dtype_code(dtype), (batch, length, hq, hk, d)
    with torch.cuda.device(device_index):  # (the workspace depends on the device's compute units)
        nbytes = _lib.attn_lib().pbattn_fp4_decode_workspace_size(*sizes)
    return sizes, code, *_window_args(window, sinks), nbytes


def _decode(q, cache, page_table, lengths, scale, window, sinks, out=None, return_lse=False):
    dev = _one_device(q, *cache, page_table, lengths)
    shape, steps, at = _fp4(cache)
    sizes, code, window, sinks, nbytes = _decode_plan(
        q.shape, q.dtype, shape, page_table.shape, lengths.shape, None if window is None else int(window), int(sinks),
        dev.index)
    q = _aligned(q.contiguous(), 16)
    page_table, lengths = _boundaries(page_table), _boundaries(lengths)
    out = _output(out, q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if return_lse else None
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch("pbattn_fp4_decode", _lib.attn_lib().pbattn_fp4_decode, dev, q.data_ptr(), code, *at, steps, shape[1], shape[0],
            page_table.data_ptr(), page_table.shape[1], lengths.data_ptr(), out.data_ptr(), _lib.ptr(lse), *sizes,
            float(scale), window, sinks, workspace.data_ptr(), nbytes)
    return out, lse


@torch.library.custom_op("pbgdn::paged_decode_attention_fp4", mutates_args=(),
                         schema="(Tensor q, Tensor k, Tensor v, Tensor k_scale, Tensor v_scale, Tensor page_table, "
                                "Tensor lengths, float scale, int? window, int sinks) -> (Tensor, Tensor)")
def paged_decode_attention_fp4_op(q, k, v, k_scale, v_scale, page_table, lengths, scale, window, sinks):
    """(o, lse) of paged_decode_attention_fp4."""
    return _decode(q, (k, v, k_scale, v_scale), page_table, lengths, scale, window, sinks, return_lse=True)


@paged_decode_attention_fp4_op.register_fake
def _(q, k, v, k_scale, v_scale, page_table, lengths, scale, window, sinks):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


def paged_decode_attention_fp4(q, cache, page_table, lengths, scale: float, window=None, sinks: int = 0, *,
                               return_lse: bool = False, out: torch.Tensor | None = None):
    """paged_decode_attention over a 4-bit cache (k, v, k_scale, v_scale): q [B,T,Hq,D] in
    float32, bfloat16 or float16, the T newest tokens of each sequence, against the values
    that the cache stands for; page_table, lengths, window, sinks, return_lse and out as
    there. Results are as exact as q's own type: softmax weights enter the products with 16 bits
    for a 16-bit q and with all of float32's 24 for a float32 one, sums are float32, and the
    result is rounded once."""
    _inference_only("paged_decode_attention_fp4", q)
    if _untraced(q, *cache, page_table, lengths):
        o, lse = _decode(q, cache, page_table, lengths, scale, window, sinks, out, return_lse)
    else:
        window = None if window is None else int(window)
        o, lse = paged_decode_attention_fp4_op(q, *cache, page_table, lengths, float(scale), window, int(sinks))
        if out is not None:
            if out.shape != o.shape or out.dtype != o.dtype:
                raise ValueError("out must have q's shape and dtype")
            o = out.copy_(o)
    return (o, lse) if return_lse else o


# ----------------------------------------------------------------------------
# Writing and reading back.
# ----------------------------------------------------------------------------
def _write(k, v, cache, slots):
    dev = _one_device(k, v, *cache, slots)
    shape, steps, at = _fp4(cache)
    code = _dtype_code(k.dtype)
    if slots.dtype not in (torch.int32, torch.int64):
        raise ValueError("slots must be int32 or int64")
    if slots.numel() >= 2**31:
        raise ValueError("paged_cache_write_fp4 takes less than 2^31 tokens")
    k, v, kv_steps = _write_operands(k, v, shape, k.dtype, slots.shape)
    if slots.dtype != torch.int64 or slots.ndim != 1 or not slots.is_contiguous():
        slots = slots.reshape(-1).to(torch.int64).contiguous()
    _launch("pbattn_fp4_write", _lib.attn_lib().pbattn_fp4_write, dev, k.data_ptr(), v.data_ptr(), code, kv_steps, *at,
            steps, shape[1], shape[0], slots.data_ptr(), slots.shape[0], shape[2], shape[3])


@torch.library.custom_op("pbgdn::paged_cache_write_fp4_", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"),
                         schema="(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
                                "Tensor(d!) v_scale, Tensor slots) -> ()")
def paged_cache_write_fp4_op(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    """paged_cache_write_fp4, for graphs of ops."""
    _write(k, v, (k_cache, v_cache, k_scale, v_scale), slots)


@paged_cache_write_fp4_op.register_fake
def _(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    return None


def paged_cache_write_fp4(k, v, cache, slots) -> None:
    """Write keys and values k, v [..., Hk, D] (float32, bfloat16 or float16; v is cast to k's
    dtype) into the pages of a 4-bit cache (k, v, k_scale, v_scale) in place: the token at
    slots[...] = s goes to row s % page of page s // page. A slot outside the cache (e.g. -1
    for padding) is skipped; the others must be distinct. Inference only."""
    _inference_only("paged_cache_write_fp4", k, v)
    if _untraced(k, v, *cache, slots):
        _write(k, v, cache, slots)
        _increment_version(tuple(cache))  # (as the op does)
    else:
        paged_cache_write_fp4_op(k, v, *cache, slots)


@_plan
def _read_plan(cache, table, lengths, tokens: int, dtype):
    """The checked code of `dtype` for a read of these shapes."""
    if len(table) != 2 or lengths != table[:1] or table[1] >= 2**31:
        raise ValueError("expected page_table [B, max_pages] and lengths [B]")
    if table[0] > MAX_REQUESTS:
        raise ValueError(f"paged_cache_read_fp4 takes at most {MAX_REQUESTS} sequences, got {table[0]}")
    if not 0 <= tokens < 2**31:
        raise ValueError("tokens must be a number of rows below 2^31")
    return _dtype_code(dtype)


def _read(cache, page_table, lengths, tokens, dtype):
    dev = _one_device(*cache, page_table, lengths)
    shape, steps, at = _fp4(cache)
    code = _read_plan(shape, page_table.shape, lengths.shape, int(tokens), dtype)
    page_table, lengths = _boundaries(page_table), _boundaries(lengths)
    k, v = (torch.empty(tokens, *shape[2:], dtype=dtype, device=dev) for _ in range(2))
    cu = lengths.new_empty(lengths.shape[0] + 1)
    _launch("pbattn_fp4_read", _lib.attn_lib().pbattn_fp4_read, dev, *at, steps, shape[1], shape[0], page_table.data_ptr(),
            page_table.shape[1], lengths.data_ptr(), k.data_ptr(), v.data_ptr(), code, cu.data_ptr(), lengths.shape[0],
            tokens, shape[2], shape[3])
    return k, v, cu


@torch.library.custom_op("pbgdn::paged_cache_read_fp4", mutates_args=(),
                         schema="(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor page_table, "
                                "Tensor lengths, int tokens, ScalarType dtype) -> (Tensor, Tensor, Tensor)")
def paged_cache_read_fp4_op(k_cache, v_cache, k_scale, v_scale, page_table, lengths, tokens, dtype):
    """paged_cache_read_fp4, for graphs of ops."""
    return _read((k_cache, v_cache, k_scale, v_scale), page_table, lengths, tokens, dtype)


@paged_cache_read_fp4_op.register_fake
def _(k_cache, v_cache, k_scale, v_scale, page_table, lengths, tokens, dtype):
    shape = (tokens, k_cache.shape[2], 2 * k_cache.shape[3])
    return (k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype),
            lengths.new_empty(lengths.shape[0] + 1, dtype=torch.int32))


def paged_cache_read_fp4(cache, page_table, lengths, tokens: int, dtype=torch.bfloat16):
    """The first lengths[b] keys and values of each sequence, packed in their order: (k, v
    [tokens, Hk, D] in `dtype`, cu_seqlens int32 [B + 1]), as window_attention takes them
    for the queries of a prompt's next piece (k[None], v[None], cu_seqlens_k=cu_seqlens).
    `tokens` is the rows' number, at least the sum of the lengths (the sequences are cut
    there); rows past the last sequence, and keys of absent pages, are zeros. bfloat16 and
    float32 hold the cache's values exactly, float16 those within its range."""
    tensors = (*cache, page_table, lengths)
    return (_read if _untraced(*tensors) else _read_traced)(cache, page_table, lengths, int(tokens), dtype)


def _read_traced(cache, page_table, lengths, tokens, dtype):
    return paged_cache_read_fp4_op(*cache, page_table, lengths, tokens, dtype)
