"""The pages of a paged cache, given to requests and taken back on the device: the page
tables and slots that pseudobrain_amd.attention's and pseudobrain_amd.fp4's paged
operators take, worked out from the requests' lengths without the host knowing them
(drafts accepted on the device, steps replayed as a graph).

A pool is a stack of free pages: free_pages int32 [capacity], of which the first
num_free (int32 [1]) are in it. Page i of a request holds its tokens i page ..
i page + page - 1 and is entry i of its row of page_table.

  paged_cache_extend   pages, slots and positions for the requests' new tokens
  paged_cache_release  pages whose tokens are no longer needed back to the pool

Which pages a request holds follows from its length. A length that is lowered, as by drafted
tokens that were not accepted, leaves pages behind that the next extension would replace by
others and the pool would never see again: they are released first, from the new length to the
old one, both rounded up to whole pages,

    up = lambda n: (n + page - 1) // page * page
    num_free = paged_cache_release(page_table, up(accepted), up(lengths), free_pages, num_free, page)

Lengths, counts and num_free are read, never changed: both return the new ones, and the
same call again gives the same results. On the GPU only; a missing library or a CPU
tensor raises.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _boundaries, _increment_version, _launch, _one_device, _plan, _untraced
from .fp4 import MAX_REQUESTS


@_plan
def _pool_plan(table, stride, dtypes, a, b, free, free_stride, num_free, page: int):
    """Checked sizes (row stride, max_pages, B, capacity) of a call with tensors of these shapes."""
    if len(table) != 2 or a != table[:1] or b != a:
        raise ValueError("expected page_table [B, max_pages] and a number for each of its B requests")
    if len(free) != 1 or num_free != (1,) or free[0] >= 2**31:
        raise ValueError("expected free_pages [capacity] and num_free [1]")
    if dtypes != (torch.int32, torch.int32):
        raise ValueError("page_table and free_pages are written in place: both must be int32")
    if (table[1] > 1 and stride[1] != 1) or (table[0] > 1 and stride[0] < table[1]) or (free[0] > 1 and free_stride[0] != 1):
        raise ValueError("page_table must have dense rows that do not overlap, free_pages be dense")
    if table[0] > MAX_REQUESTS:
        raise ValueError(f"the pool takes at most {MAX_REQUESTS} requests at once, got {table[0]}")
    if page < 1:
        raise ValueError("a page holds at least one token")
    if table[1] * page >= 2**31:
        raise ValueError("a request's pages must hold less than 2^31 tokens")
    return (stride[0] if table[0] > 1 else table[1]), table[1], table[0], free[0]


def _pool(page_table, a, b, free_pages, num_free, page):
    """The device, _pool_plan's sizes, and the three integer tensors as the kernels read them."""
    dev = _one_device(page_table, a, b, free_pages, num_free)
    sizes = _pool_plan(page_table.shape, page_table.stride(), (page_table.dtype, free_pages.dtype), a.shape, b.shape,
                       free_pages.shape, free_pages.stride(), num_free.shape, page)
    return dev, sizes, _boundaries(a), _boundaries(b), _boundaries(num_free)


def _extend(page_table, lengths, counts, free_pages, num_free, page, tokens):
    dev, (row, max_pages, batch, capacity), lengths, counts, num_free = _pool(
        page_table, lengths, counts, free_pages, num_free, page)
    if not 0 <= tokens < 2**31:
        raise ValueError("tokens must be a number of tokens below 2^31")
    slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    positions, cu, new_lengths, new_free = [lengths.new_empty(n) for n in (tokens, batch + 1, batch, 1)]
    _launch("pbattn_pages_extend", _lib.attn_lib().pbattn_pages_extend, dev, page_table.data_ptr(), row, max_pages,
            lengths.data_ptr(), counts.data_ptr(), batch, page, free_pages.data_ptr(), capacity, num_free.data_ptr(), tokens,
            slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), new_lengths.data_ptr(), new_free.data_ptr())
    return slots, positions, cu, new_lengths, new_free


@torch.library.custom_op("pbgdn::paged_cache_extend_", mutates_args=("page_table",),
                         schema="(Tensor(a!) page_table, Tensor lengths, Tensor counts, Tensor free_pages, "
                                "Tensor num_free, int page, int tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
def paged_cache_extend_op(page_table, lengths, counts, free_pages, num_free, page, tokens):
    """paged_cache_extend, for graphs of ops."""
    return _extend(page_table, lengths, counts, free_pages, num_free, page, tokens)


@paged_cache_extend_op.register_fake
def _(page_table, lengths, counts, free_pages, num_free, page, tokens):
    batch = lengths.shape[0]
    return (lengths.new_empty(tokens, dtype=torch.int64),
            *(lengths.new_empty(n, dtype=torch.int32) for n in (tokens, batch + 1, batch, 1)))


def paged_cache_extend(page_table, lengths, counts, free_pages, num_free, page: int, tokens: int):
    """Places for the requests' new tokens: request b, with lengths[b] tokens in the cache,
    gets counts[b] more (int [B] both; none where it is not positive), and the pages they
    need from the top of the pool, which are entered in page_table [B, max_pages] in place.

    Requests are gone through in order; one gets all it asks for or nothing. It is granted
    if its tokens and all asked for before it are at most `tokens`, if they fit its row of the
    table, and if the pool holds the pages wanted up to it (or it wants none). Returns

      slots        int64 [tokens]: the granted tokens' slots, packed in the requests'
                   order (as paged_cache_write takes them), -1 past the last
      positions    int32 [tokens]: each token's place in its request, -1 past the last
                   (as qk_norm_rope takes them)
      cu_seqlens   int32 [B + 1]: where each request's new tokens start and end
      lengths      int32 [B]: with the tokens granted (as paged_decode_attention takes them)
      num_free     int32 [1]: pages left

    A request's place that is not granted shows as an unchanged length; ask again once pages
    have been released. Pages past lengths[b] count as not held: where a length was lowered they
    have to be released before (see the module)."""
    args = (page_table, lengths, counts, free_pages, num_free)
    if not _untraced(*args):
        return paged_cache_extend_op(*args, int(page), int(tokens))
    out = _extend(*args, int(page), int(tokens))
    _increment_version(page_table)  # (as the op does)
    return out


def _release(page_table, first, end, free_pages, num_free, page):
    dev, (row, max_pages, batch, capacity), first, end, num_free = _pool(page_table, first, end, free_pages, num_free, page)
    new_free = first.new_empty(1)
    _launch("pbattn_pages_release", _lib.attn_lib().pbattn_pages_release, dev, page_table.data_ptr(), row, max_pages,
            first.data_ptr(), end.data_ptr(), batch, page, free_pages.data_ptr(), capacity, num_free.data_ptr(),
            new_free.data_ptr())
    return new_free


@torch.library.custom_op("pbgdn::paged_cache_release_", mutates_args=("free_pages",),
                         schema="(Tensor page_table, Tensor first, Tensor end, Tensor(a!) free_pages, Tensor num_free, "
                                "int page) -> Tensor")
def paged_cache_release_op(page_table, first, end, free_pages, num_free, page):
    """paged_cache_release, for graphs of ops."""
    return _release(page_table, first, end, free_pages, num_free, page)


@paged_cache_release_op.register_fake
def _(page_table, first, end, free_pages, num_free, page):
    return first.new_empty(1, dtype=torch.int32)


def paged_cache_release(page_table, first, end, free_pages, num_free, page: int):
    """Give pages back: those of request b whose last token lies in [first[b], end[b]) (int
    [B] both) are pushed on the pool, free_pages in place, in the requests' order; entries
    below 0 are no pages and are left out. Returns the new num_free, int32 [1]; page_table
    stays as it is.

    Ranges that follow each other give every page back once: a window's, as it moves on
    (first no less than the sinks' pages times `page`), from behind, as a length is lowered
    (both ends rounded up to whole pages), and in the end the rest, end rounded up to a whole
    page. A page must not be given back twice."""
    args = (page_table, first, end, free_pages, num_free)
    if not _untraced(*args):
        return paged_cache_release_op(*args, int(page))
    out = _release(*args, int(page))
    _increment_version(free_pages)  # (as the op does)
    return out
