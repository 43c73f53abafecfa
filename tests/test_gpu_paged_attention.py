"""paged_decode_attention and paged_cache_write on the device: against the float64
oracle (oracle/attention.py) within its error bounds, and the cache bit for bit."""
import numpy as np
import pytest
import torch

from oracle import attention as oa
from pseudobrain_amd import attention as at
from tests.test_gpu_window_attention import NAMES, compare, f64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lengths, page, hq, hk, d, draft, dtype, seed, heads_first=False, spare=3):
    """Caches with shuffled pages, a table without entries past each length."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    kc, vc = (torch.randn(shape, generator=gen).to(dtype).to(DEV) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    perm = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[first:first + n]
        first += n
    q = torch.randn(len(lengths), draft, hq, d, generator=gen).to(dtype).to(DEV)
    return q, kc, vc, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def rows(cache, table, b, n):
    """The first n cached rows of sequence b, float64 [n, Hk, D]."""
    page = cache.shape[1]
    index = table[b, :-(-n // page)].long()
    return f64(cache[index].reshape(-1, *cache.shape[2:])[:n])


def check(where, q, kc, vc, table, lengths, scale, window=None, sinks=0):
    print(f"[{where}] q {tuple(q.shape)} cache {tuple(kc.shape)} window {window} sinks {sinks} {q.dtype}", flush=True)
    o, lse = at.paged_decode_attention(q, kc, vc, table, lengths, scale, window, sinks, return_lse=True)
    torch.cuda.synchronize()
    refs = []
    for b, n in enumerate(lengths.tolist()):
        n = max(n, 0)
        refs.append(oa.attention(f64(q[b]), rows(kc, table, b, n), rows(vc, table, b, n), scale, window, sinks,
                                 dtype=NAMES[q.dtype]))
    compare(where + " o", o, np.stack([r["o"] for r in refs]), np.stack([r["o_tol"] for r in refs]))
    compare(where + " lse", lse, np.stack([r["lse"] for r in refs]), np.stack([r["lse_tol"] for r in refs]))
    return o, lse


@pytest.mark.parametrize("page", [1, 7, 16, 100, 528])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (40, 5), (600, 64)])
def test_pages_windows_and_lengths(page, window, sinks):
    """Lengths of zero, one and around the blocks; pages that end inside them."""
    x = make([0, 1, 31, 32, 33, 127, 129, 700, 1300, -4], page, 8, 2, 128, 1, torch.bfloat16, page)
    o, lse = check("pages", *x, 128 ** -0.5, window, sinks)
    for b in (0, 9):
        assert torch.count_nonzero(o[b]) == 0 and torch.isneginf(lse[b]).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths_and_types(d, dtype):
    for draft, hq in ((1, 4), (3, 16)):
        x = make([300, 5, 1000], 16, hq, 2, d, draft, dtype, d)
        check(f"widths draft {draft}", *x, d ** -0.5, 200, 3)


@pytest.mark.parametrize("hq,hk,draft", [(1, 1, 1), (3, 3, 2), (7, 1, 1), (16, 1, 1), (17, 1, 1), (40, 1, 1), (6, 2, 5),
                                         (8, 1, 16), (24, 8, 4)])
def test_head_groups_and_drafts(hq, hk, draft):
    """Rows that fill one matrix tile, two, and more than a workgroup's; drafts
    longer than their sequence see nothing."""
    x = make([400, 33, draft, 1, 2], 16, hq, hk, 64, draft, torch.bfloat16, hq + draft)
    check("groups", *x, 0.125)
    check("groups, window", *x, 0.125, 20, 2)


def test_long_contexts_are_split_and_joined():
    x = make([20000, 3, 9000], 64, 8, 1, 128, 1, torch.bfloat16, 20)
    check("split", *x, 128 ** -0.5)
    x = make([20000, 3, 9000], 64, 4, 1, 64, 2, torch.float32, 21)
    check("split float32", *x, 0.125)


def test_large_batches():
    lengths = [(i * 37) % 200 for i in range(300)]
    x = make(lengths, 16, 4, 2, 64, 1, torch.bfloat16, 22)
    check("batch of 300", *x, 0.125)


def test_cache_layouts():
    """Heads before tokens in a page, and keys and values interleaved by page."""
    x = make([100, 260], 16, 4, 2, 64, 1, torch.bfloat16, 23, heads_first=True)
    check("heads first", *x, 0.125, 50, 3)
    q, kc, vc, table, lengths = make([100, 260], 16, 4, 2, 64, 1, torch.bfloat16, 24)
    both = torch.stack((kc, vc), 1)
    check("interleaved", q, both[:, 0], both[:, 1], table, lengths, 0.125, 50, 3)


def test_absent_pages_and_stale_rows():
    """Entries that no query sees may be anything; the keys of an entry outside
    the cache are absent; rows past the length and unused pages hold NaN."""
    q, kc, vc, table, lengths = make([500, 90], 16, 4, 2, 64, 1, torch.bfloat16, 25)
    want = at.paged_decode_attention(q, kc, vc, table, lengths, 0.125, 64, 4)
    used = torch.zeros(kc.shape[0], dtype=torch.bool)
    freed = table.clone()
    freed[0, 1:(500 - 64) // 16] = torch.tensor([-1, 10 ** 6] * 20, dtype=torch.int32, device=DEV)[:(500 - 64) // 16 - 1]
    for b, n in enumerate([500, 90]):
        for i in range(-(-n // 16)):
            if 0 <= freed[b, i] < kc.shape[0]:
                used[freed[b, i]] = True
    for cache in (kc, vc):
        cache[~used.to(DEV)] = float("nan")
        cache[table[0, 500 // 16].long(), 500 % 16:] = float("nan")
        cache[table[1, 90 // 16].long(), 90 % 16:] = float("inf")
    got = at.paged_decode_attention(q, kc, vc, freed, lengths, 0.125, 64, 4)
    assert torch.equal(got, want)
    # an absent page in the window: as if its keys did not exist
    kc, vc = torch.nan_to_num(kc, 0, 0, 0), torch.nan_to_num(vc, 0, 0, 0)
    hole = table.clone()
    hole[1, 2] = -1
    o = at.paged_decode_attention(q, kc, vc, hole, lengths, 0.125)
    k, v = rows(kc, table, 1, 90), rows(vc, table, 1, 90)
    keep = np.r_[0:32, 48:90]
    ref = oa.attention(f64(q[1]), k[keep], v[keep], 0.125, dtype="bfloat16")
    compare("hole", o[1], ref["o"], ref["o_tol"])
    # a length beyond the table, and no pages at all
    longer = at.paged_decode_attention(q, kc, vc, table[:, :6].contiguous(), torch.tensor([5000, 90], device=DEV,
                                                                                         dtype=torch.int32), 0.125)
    assert torch.isfinite(longer).all()
    none = at.paged_decode_attention(q, kc[:0], vc[:0], table, lengths, 0.125)
    assert torch.count_nonzero(none) == 0


@pytest.mark.parametrize("d,dtype", [(64, torch.float32), (64, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16),
                                     (256, torch.float32)])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_a_bad_value_reaches_only_the_tokens_that_see_it(d, dtype, group):
    """Infinities and NaN among the drafts and at the window's edge, in values and keys."""
    draft, window, lengths = 4, 50, [200, 131]
    q, kc, vc, table, lens = make(lengths, 16, 2 * group, 2, d, draft, dtype, 31)
    clean = at.paged_decode_attention(q, kc, vc, table, lens, d ** -0.5, window, 3)
    bad = {0: (200 - 1, 200 - 4 - window + 1, 200 - 2), 1: (131 - 2, 131 - 4 - window + 2, 131 - 1)}
    for b, (x, y, key) in bad.items():
        vc[table[b, x // 16].long(), x % 16, :, 3] = float("inf")
        vc[table[b, y // 16].long(), y % 16, :, 5] = float("nan")
        kc[table[b, key // 16].long(), key % 16] = float("nan")
    got, lse = at.paged_decode_attention(q, kc, vc, table, lens, d ** -0.5, window, 3, return_lse=True)
    # both sides within a bound of u (|o| + sum p |v|) of the truth, values up to 6
    bound = 4 * 6 * oa.UNIT[NAMES[dtype]] + 1e-4
    for b, (x, y, key) in bad.items():
        for t in range(draft):
            pos = lengths[b] - draft + t
            sees_x, sees_y, sees_key = (pos - window < j <= pos for j in (x, y, key))
            if sees_key:
                assert torch.isnan(got[b, t]).all()
                continue
            assert torch.isfinite(lse[b, t]).all()
            hit = torch.zeros(d, dtype=torch.bool, device=DEV)
            hit[3], hit[5] = sees_x, sees_y
            assert not torch.isfinite(got[b, t][:, hit]).any()
            assert (got[b, t][:, ~hit].float() - clean[b, t][:, ~hit].float()).abs().max() <= bound


def test_offsets_past_32_bits():
    """Rows of a cache beyond 4 GiB (keys and values each)."""
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GiB of free device memory")
    pages, page, hk, d = 4200, 16, 128, 256  # 4.4 GB each in bfloat16
    kc, vc = (torch.zeros(pages, page, hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    torch.manual_seed(26)
    k, v = (torch.randn(40, hk, d, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = (pages - 3) * page + torch.arange(40, device=DEV)
    at.paged_cache_write(k, v, kc, vc, slots)
    assert torch.equal(kc[pages - 3:].reshape(-1, hk, d)[:40], k)
    q = torch.randn(1, 1, hk, d, device=DEV).to(torch.bfloat16)
    table = torch.tensor([[pages - 3, pages - 2, pages - 1]], dtype=torch.int32, device=DEV)
    o = at.paged_decode_attention(q, kc, vc, table, torch.tensor([40], dtype=torch.int32, device=DEV), 0.0625)
    ref = oa.attention(f64(q[0]), f64(k), f64(v), 0.0625, dtype="bfloat16")
    compare("past 32 bits", o[0], ref["o"], ref["o_tol"])


def test_equal_runs_and_graph_replay():
    """Captured and replayed several times among eager work, each replay bit-equal."""
    q, kc, vc, table, lengths = make([3000, 17, 900, 0], 16, 8, 2, 128, 1, torch.bfloat16, 27)
    k, v = (torch.randn(4, 2, 128, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([table[0, 2999 // 16].item() * 16 + 2999 % 16, -1, 10 ** 9, -7], device=DEV)

    def step():
        at.paged_cache_write(k, v, kc, vc, slots)
        return at.paged_decode_attention(q, kc, vc, table, lengths, 0.09, 500, 4)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(step(), want)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 256), (torch.bfloat16, 72)])
def test_cache_write(dtype, d):
    """Rows land where their slots say, skipped slots and all other rows stay."""
    gen = torch.Generator().manual_seed(28)
    pages, page, hk, n = 9, 13, 3, 70
    for heads_first in (False, True):
        shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
        kc, vc = (torch.randn(shape, generator=gen).to(dtype).to(DEV) for _ in range(2))
        if heads_first:
            kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
        kv = torch.randn(n, 2 * hk * d, generator=gen).to(dtype).to(DEV)
        k, v = (x.view(n, hk, d) for x in kv.split(hk * d, -1))  # strided rows
        slots = torch.randperm(pages * page, generator=gen)[:n]
        slots[5], slots[17], slots[40] = -1, pages * page, 2 ** 40
        want = [c.clone().reshape(-1, hk, d) for c in (kc, vc)]
        for w, x in zip(want, (k, v)):
            keep = (slots >= 0) & (slots < pages * page)
            w[slots[keep].to(DEV)] = x[keep.to(DEV)]
        at.paged_cache_write(k, v, kc, vc, slots.to(DEV))
        for c, w in zip((kc, vc), want):
            assert torch.equal(c.reshape(-1, hk, d), w)
    # leading axes, int32 slots and another dtype of the new rows
    k4, v4 = (torch.randn(2, 3, hk, d, generator=gen).to(DEV) for _ in range(2))
    slots = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    at.paged_cache_write(k4, v4, kc, vc, slots)
    assert torch.equal(kc[0, :6], k4.view(6, hk, d).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cache_write_of_column_slices_off_the_alignment(dtype):
    """New rows as columns of wider rows, 8 bytes off the alignment."""
    skip, pad, n, hk, d = 8 // dtype.itemsize, 16 // dtype.itemsize, 30, 2, 64
    torch.manual_seed(30)
    k, v = (torch.randn(n, hk * d + pad, device=DEV).to(dtype)[:, skip:skip + hk * d].unflatten(-1, (hk, d))
            for _ in range(2))
    assert k.data_ptr() % 16 == 8
    kc, vc = (torch.zeros(4, 8, hk, d, dtype=dtype, device=DEV) for _ in range(2))
    at.paged_cache_write(k, v, kc, vc, torch.arange(n, device=DEV))
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c.view(-1, hk, d)[:n], x) and torch.count_nonzero(c.view(-1, hk, d)[n:]) == 0


def test_prefill_then_decode_equals_one_pass():
    """A prompt attended and cached, then tokens one at a time, against window_attention over all of it."""
    torch.manual_seed(29)
    n, extra, hq, hk, d, page, window, sinks = 150, 40, 8, 2, 64, 16, 60, 4
    q, k, v = (torch.randn(1, n + extra, h, d, device=DEV).to(torch.bfloat16) for h in (hq, hk, hk))
    whole, lse = at.window_attention(q, k, v, 0.125, window, sinks, return_lse=True)
    kc, vc = (torch.full((20, page, hk, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.randperm(20, device=DEV).to(torch.int32)[None]
    slot = lambda j: table[0, j // page].long() * page + j % page  # noqa: E731
    at.paged_cache_write(k[0, :n], v[0, :n], kc, vc, slot(torch.arange(n, device=DEV)))
    for t in range(n, n + extra):
        at.paged_cache_write(k[0, t:t + 1], v[0, t:t + 1], kc, vc, slot(torch.tensor([t], device=DEV)))
        o, l1 = at.paged_decode_attention(q[:, t:t + 1], kc, vc, table, torch.tensor([t + 1], dtype=torch.int32,
                                                                                      device=DEV), 0.125, window, sinks,
                                          return_lse=True)
        # two roundings of p and o to bfloat16 over values of size 4 at most
        torch.testing.assert_close(o.float(), whole[:, t:t + 1].float(), rtol=0, atol=4 * 4 * 2.0 ** -8)
        torch.testing.assert_close(l1, lse[:, t:t + 1], rtol=0, atol=1e-4)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.bfloat16, 256)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("scale", [1.0, 4.0])
@pytest.mark.parametrize("draft,hq", [(1, 2), (3, 16)])
def test_scores_at_the_ends_of_the_range(dtype, d, sign, scale, draft, hq):
    """Equal scores of 3.3e38 or its negative, in one part and in parts that are joined: means of the values."""
    lengths = [40, 9000, 700]
    q, kc, vc, table, lens = make(lengths, 16, hq, 2, d, draft, dtype, 39)
    q.zero_(), kc.zero_()
    q[..., 0], kc[..., 0] = 1.0, sign * 3.3e38
    o, lse = at.paged_decode_attention(q, kc, vc, table, lens, scale, return_lse=True)
    want = min(3.3e38 * scale, torch.finfo(torch.float32).max) * sign
    assert torch.isfinite(lse).all() and (lse.double() - want).abs().max() <= 2 ** -7 * abs(want)
    for b, n in enumerate(lengths):
        v = rows(vc, table, b, n)
        for t in range(draft):
            mean = v[:n - draft + 1 + t].mean(0).repeat(hq // 2, 0)
            u = max(oa.UNIT[NAMES[dtype]], n * 2.0 ** -24)
            assert (np.abs(f64(o[b, t]) - mean) <= 4 * u * np.abs(v).max()).all()


def test_compiled_decoding_equals_eager():
    """A decode step under torch.compile: the caches and outputs of the eager calls, no break in the graph."""
    q, kc, vc, table, lengths = make([300, 17, 90], 16, 8, 2, 64, 1, torch.bfloat16, 32)
    k, v = (torch.randn(3, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = torch.stack([table[b, (n - 1) // 16] * 16 + (n - 1) % 16 for b, n in enumerate((300, 17, 90))]).long()

    def step(q, k, v, kc, vc, slots, out=None):
        at.paged_cache_write(k, v, kc, vc, slots)
        return at.paged_decode_attention(q * 2, kc, vc, table, lengths, 0.125, 50, 3, out=out) + 1

    other = kc.clone(), vc.clone()
    with torch.no_grad():
        compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
        want = step(q, k, v, kc, vc, slots)
        assert torch.equal(compiled(q, k, v, *other, slots), want)
        assert torch.equal(other[0], kc) and torch.equal(other[1], vc)
        outs = [torch.zeros_like(q) for _ in range(2)]
        assert torch.equal(compiled(q, k, v, *other, slots, outs[0]), step(q, k, v, kc, vc, slots, outs[1]))
        assert torch.equal(*outs)


def test_paged_ops_pass_the_opcheck():
    q, kc, vc, table, lengths = make([30, 7], 16, 4, 2, 64, 1, torch.float32, 33)
    k, v = (torch.randn(2, 2, 64, device=DEV) for _ in range(2))
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(at.paged_decode_attention_op, (q, kc, vc, table, lengths, 0.125, 8, 1), test_utils=utils)
    torch.library.opcheck(at.paged_cache_write_op, (k, v, kc, vc, torch.tensor([3, 20], device=DEV)), test_utils=utils)
