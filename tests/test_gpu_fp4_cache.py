"""The 4-bit cache on the device: writes and reads bit for bit against the format's
definition (oracle/fp4.py), decoding over it against float64 attention of the values
that it stands for (oracle/attention.py), within that oracle's error bounds."""
import numpy as np
import pytest
import torch

from oracle import attention as oa
from oracle import fp4 as of
from pseudobrain_amd import _lib
from pseudobrain_amd import attention as at
from pseudobrain_amd import fp4 as fc
from pseudobrain_amd.workloads import to_numpy
from tests.test_gpu_window_attention import NAMES, compare, f64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def filled(pages, page, heads, width, seed, heads_first=False, spread=2):
    """A cache of random codes, scales 2^-spread .. 2^spread."""
    gen = torch.Generator().manual_seed(seed)
    cache = fc.fp4_cache(pages, page, heads, width, DEV, heads_first)
    for x in cache[:2]:
        x.copy_(torch.randint(256, x.shape, generator=gen).to(torch.uint8))
    for x in cache[2:]:
        x.copy_(torch.randint(127 - spread, 128 + spread, x.shape, generator=gen).to(torch.uint8))
    return cache


def make(lengths, page, hq, hk, d, draft, dtype, seed, heads_first=False, spare=3):
    """A cache with shuffled pages, a table without entries past each length."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[first:first + n]
        first += n
    q = torch.randn(len(lengths), draft, hq, d, generator=gen).to(dtype).to(DEV)
    cache = filled(pages, page, hk, d, seed + 1, heads_first)
    return q, cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def held(data, scales):
    return of.values(to_numpy(data), to_numpy(scales))


def rows(cache, table, b, n):
    """The first n cached keys and values of sequence b, float64 [n, Hk, D]."""
    page = cache[0].shape[1]
    index = table[b, :-(-n // page)].long()
    return [held(cache[i][index], cache[2 + i][index]).reshape(-1, cache[0].shape[2], 2 * cache[0].shape[3])[:n]
            for i in range(2)]


def check(where, q, cache, table, lengths, scale, window=None, sinks=0):
    print(f"[{where}] q {tuple(q.shape)} codes {tuple(cache[0].shape)} window {window} sinks {sinks} {q.dtype}", flush=True)
    o, lse = fc.paged_decode_attention_fp4(q, cache, table, lengths, scale, window, sinks, return_lse=True)
    torch.cuda.synchronize()
    refs = []
    for b, n in enumerate(lengths.tolist()):
        refs.append(oa.attention(f64(q[b]), *rows(cache, table, b, max(n, 0)), scale, window, sinks, dtype=NAMES[q.dtype]))
    compare(where + " o", o, np.stack([r["o"] for r in refs]), np.stack([r["o_tol"] for r in refs]))
    compare(where + " lse", lse, np.stack([r["lse"] for r in refs]), np.stack([r["lse_tol"] for r in refs]))
    return o, lse


# ----------------------------------------------------------------------------
# Decoding.
# ----------------------------------------------------------------------------
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
@pytest.mark.parametrize("heads_first", [False, True])
def test_widths_and_types(d, dtype, heads_first):
    for draft, hq in ((1, 4), (3, 16)):
        x = make([300, 5, 1000], 16, hq, 2, d, draft, dtype, d, heads_first)
        check(f"widths draft {draft}", *x, d ** -0.5, 200, 3)
        check(f"widths draft {draft}, scale < 0", *x, -(d ** -0.5))


@pytest.mark.parametrize("hq,hk,draft", [(1, 1, 1), (3, 3, 2), (7, 1, 1), (16, 1, 1), (17, 1, 1), (40, 1, 1), (6, 2, 5),
                                         (8, 1, 16), (24, 8, 4)])
def test_head_groups_and_drafts(hq, hk, draft):
    """Rows that fill one matrix tile, two, and more than a workgroup's; drafts
    longer than their sequence see nothing."""
    x = make([400, 33, draft, 1, 2], 16, hq, hk, 64, draft, torch.bfloat16, hq + draft)
    check("groups", *x, 0.125)
    check("groups, window", *x, 0.125, 20, 2)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("draft,hq", [(1, 4), (3, 16)])
def test_a_result_is_rounded_once(d, dtype, draft, hq):
    """Weights do not lose the bits that a result of q's type can show: they enter the products in
    two parts of 16 bits (off by less than 2^-15 of themselves), for float32 rows in three, all
    of their bits. So the bound is a float32 kernel's (oracle/attention.py), 2^-15 of the sum of
    magnitudes, and one rounding of the result."""
    q, cache, table, lengths = make([300, 5, 1000], 16, hq, 2, d, draft, dtype, d + 3)
    o = fc.paged_decode_attention_fp4(q, cache, table, lengths, d ** -0.5, 200, 3)
    u, cut = (0.0, 0.0) if dtype == torch.float32 else (oa.UNIT[NAMES[dtype]], 2.0 ** -15)
    for b, n in enumerate(lengths.tolist()):
        k, v = rows(cache, table, b, n)
        ref = oa.attention(f64(q[b]), k, v, d ** -0.5, 200, 3)
        size = oa.attention(f64(q[b]), k, np.abs(v), d ** -0.5, 200, 3)["o"]
        tol = ref["o_tol"] + u * np.abs(ref["o"]) + 1.01 * cut * size + oa.TINY[NAMES[dtype]]
        compare(f"rounded once, {n}", o[b], ref["o"], tol)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weights_are_rounded_to_nearest(d, dtype):
    """Six keys of weight 1 and value 1, eleven of weight 6 / 11 and value -1: their sum is what
    the weights lose. 6 / 11 has 0.909 steps of 2^-16 behind its 16 bits: cut off they would leave
    11 / 12 0.909 2^-16 = 1.27e-5 of the output; rounded to nearest, a weight is off by at most
    2^-17, the output by 11 / 12 of that, and by 2^-19 for float32 arithmetic on 17 terms (17
    2^-24 at most) and the exponential (2^-21 and less)."""
    q, cache, table, lengths = make([17], 32, 1, 1, d, 1, dtype, d)
    q.zero_()
    for x in cache[:2]:
        x.zero_()
    for x in cache[2:]:
        x.fill_(127)
    q[..., 0] = -1.0
    page = table[0, 0].item()
    cache.k[page, 6:17, 0, 0] = 0x02  # 1 in the row's first value: a score of -scale
    cache.v[page, :6], cache.v[page, 6:17] = 0x22, 0xaa  # 1 and -1
    o = fc.paged_decode_attention_fp4(q, cache, table, lengths, float(np.log(11 / 6)))
    bound = (0.0 if dtype == torch.float32 else 11 / 12 * 2.0 ** -17) + 2.0 ** -19
    print(f"[weights] {np.abs(f64(o)).max():.3e} of {bound:.3e}", flush=True)
    assert np.abs(f64(o)).max() <= bound


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,draft", [(6, 3, 1), (3, 3, 5), (24, 3, 3), (7, 1, 1), (20, 1, 1)])
def test_an_odd_number_of_heads(d, dtype, hq, hk, draft):
    """Heads whose rows share lines with the next one's, and one head alone."""
    for heads_first, page in ((False, 16), (True, 2)):
        x = make([300, 5, 1000], page, hq, hk, d, draft, dtype, d + hk, heads_first)
        check("odd heads", *x, d ** -0.5, 400, 3)


def test_long_contexts_are_split_and_joined():
    x = make([20000, 3, 9000], 64, 8, 1, 128, 1, torch.bfloat16, 20)
    check("split", *x, 128 ** -0.5)
    x = make([20000, 3, 9000], 64, 4, 1, 64, 2, torch.float32, 21)
    check("split float32", *x, 0.125)


def test_large_batches():
    lengths = [(i * 37) % 200 for i in range(300)]
    x = make(lengths, 16, 4, 2, 64, 1, torch.bfloat16, 22)
    check("batch of 300", *x, 0.125)
    lengths = [(i * 37) % 23 for i in range(1500)]
    lengths[700], lengths[1499] = 3000, 1000
    x = make(lengths, 16, 4, 2, 64, 1, torch.bfloat16, 23)
    check("batch of 1500", *x, 0.125)


def test_large_and_small_rows_of_float32_and_float16():
    """Queries and scales at the ends of their types' ranges: the parts of a product add up to it."""
    for dtype, size in ((torch.float32, 1e30), (torch.float32, 1e-30), (torch.float16, 6e4), (torch.float16, 6e-6)):
        q, cache, table, lengths = make([90, 700], 16, 4, 2, 64, 1, dtype, 23)
        q = (q / q.abs().max() * size).to(dtype)
        check(f"size {size}", q, cache, table, lengths, 1.0 / size)


def test_absent_pages_and_stale_rows():
    """Entries that no query sees may be anything; the keys of an entry outside the cache
    are absent; rows past the length and unused pages hold the scale of NaN."""
    q, cache, table, lengths = make([500, 90], 16, 4, 2, 64, 1, torch.bfloat16, 25)
    want = fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.125, 64, 4)
    pages = cache.k.shape[0]
    used = torch.zeros(pages, dtype=torch.bool)
    freed = table.clone()
    freed[0, 1:(500 - 64) // 16] = torch.tensor([-1, 10 ** 6] * 20, dtype=torch.int32, device=DEV)[:(500 - 64) // 16 - 1]
    for b, n in enumerate([500, 90]):
        for i in range(-(-n // 16)):
            if 0 <= freed[b, i] < pages:
                used[freed[b, i]] = True
    for scales in cache[2:]:
        scales[~used.to(DEV)] = 255
        scales[table[0, 500 // 16].long(), 500 % 16:] = 255
        scales[table[1, 90 // 16].long(), 90 % 16:] = 255
    got = fc.paged_decode_attention_fp4(q, cache, freed, lengths, 0.125, 64, 4)
    assert torch.equal(got, want)
    # an absent page in the window: as if its keys did not exist
    hole = table.clone()
    hole[1, 2] = -1
    o = fc.paged_decode_attention_fp4(q, cache, hole, lengths, 0.125)
    k, v = rows(cache, table, 1, 90)
    keep = np.r_[0:32, 48:90]
    ref = oa.attention(f64(q[1]), k[keep], v[keep], 0.125, dtype="bfloat16")
    compare("hole", o[1], ref["o"], ref["o_tol"])
    # a length beyond the table, and no pages at all
    whole = filled(pages, 16, 2, 64, 3)
    longer = fc.paged_decode_attention_fp4(q, whole, table[:, :6].contiguous(),
                                           torch.tensor([5000, 90], device=DEV, dtype=torch.int32), 0.125)
    assert torch.isfinite(longer).all()
    none = fc.paged_decode_attention_fp4(q, tuple(x[:0] for x in cache), table, lengths, 0.125)
    assert torch.count_nonzero(none) == 0
    no_table = fc.paged_decode_attention_fp4(q, whole, table[:, :0], lengths, 0.125)
    assert torch.count_nonzero(no_table) == 0


@pytest.mark.parametrize("d,dtype", [(64, torch.float32), (64, torch.float16), (128, torch.bfloat16), (256, torch.bfloat16),
                                     (256, torch.float32)])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("heads_first", [False, True])
def test_a_bad_value_reaches_only_the_tokens_that_see_it(d, dtype, group, heads_first):
    """Scales of NaN among the drafts and at the window's edge, in values and keys."""
    draft, window, lengths = 4, 50, [200, 131]
    q, cache, table, lens = make(lengths, 16, 2 * group, 2, d, draft, dtype, 31, heads_first)
    clean = fc.paged_decode_attention_fp4(q, cache, table, lens, d ** -0.5, window, 3)
    bad = {0: (200 - 1, 200 - 4 - window + 1, 200 - 2), 1: (131 - 2, 131 - 4 - window + 2, 131 - 1)}
    for b, (x, y, key) in bad.items():
        cache.v_scale[table[b, x // 16].long(), x % 16, :, 0] = 255
        cache.v_scale[table[b, y // 16].long(), y % 16, :, 1] = 255
        cache.k_scale[table[b, key // 16].long(), key % 16] = 255
    got, lse = fc.paged_decode_attention_fp4(q, cache, table, lens, d ** -0.5, window, 3, return_lse=True)
    # both sides within a bound of u (|o| + sum p |v|) of the truth, values up to 6 2^2
    bound = 4 * 24 * oa.UNIT[NAMES[dtype]] + 1e-3
    for b, (x, y, key) in bad.items():
        for t in range(draft):
            pos = lengths[b] - draft + t
            sees_x, sees_y, sees_key = (pos - window < j <= pos for j in (x, y, key))
            if sees_key:
                assert torch.isnan(got[b, t]).all()
                continue
            assert torch.isfinite(lse[b, t]).all()
            hit = torch.zeros(d, dtype=torch.bool, device=DEV)
            hit[:32], hit[32:64] = sees_x, sees_y
            assert not torch.isfinite(got[b, t][:, hit]).any()
            assert (got[b, t][:, ~hit].float() - clean[b, t][:, ~hit].float()).abs().max() <= bound


def test_offsets_past_32_bits():
    """Codes beyond 4 GiB (keys and values each), written, read and attended."""
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GiB of free device memory")
    pages, page, hk, d = 16900, 16, 128, 256  # 4.4 GB of codes each
    for heads_first in (False, True):
        cache = fc.fp4_cache(pages, page, hk, d, DEV, heads_first)
        torch.manual_seed(26)
        k, v = (torch.randn(40, hk, d, device=DEV).to(torch.bfloat16) for _ in range(2))
        fc.paged_cache_write_fp4(k, v, cache, (pages - 3) * page + torch.arange(40, device=DEV))
        want = [of.values(*of.quantise(f64(x))) for x in (k, v)]
        table = torch.tensor([[pages - 3, pages - 2, pages - 1]], dtype=torch.int32, device=DEV)
        lengths = torch.tensor([40], dtype=torch.int32, device=DEV)
        got = fc.paged_cache_read_fp4(cache, table, lengths, 40)
        for x, w in zip(got, want):
            np.testing.assert_array_equal(f64(x), w)
        q = torch.randn(1, 1, hk, d, device=DEV).to(torch.bfloat16)
        o = fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.0625)
        ref = oa.attention(f64(q[0]), *want, 0.0625, dtype="bfloat16")
        compare("past 32 bits", o[0], ref["o"], ref["o_tol"])


def test_every_kernel_past_32_bits():
    """Decoding over codes beyond 4 GiB: each width, type and number of row tiles, pages at both ends of
    the cache, drafts, the last of which sees keys and values whose scale is that of NaN."""
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GiB of free device memory")
    pages, page, n, draft = 16900, 16, 75, 4  # 4.4 GB of codes each
    whole = fc.fp4_cache(pages, page, 128, 256, DEV, False)
    lengths = torch.tensor([n, 0], dtype=torch.int32, device=DEV)
    first = torch.tensor([pages - 1, 0, pages - 3, 1, pages - 2], dtype=torch.int32, device=DEV)
    table = torch.stack((first, first))
    slots = (first.long()[:, None] * page + torch.arange(page, device=DEV)).flatten()[:n]
    hk = 2
    for d in (64, 128, 256):
        cache = [x.view(pages, page, 128 * 256 // d, -1)[:, :, :hk] for x in whole]  # its first heads
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            gen = torch.Generator().manual_seed(d)
            k, v = (torch.randn(n, hk, d, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
            held_k, held_v = (of.values(*of.quantise(f64(x))) for x in (k, v))
            for group, t in ((3, 1), (2, draft), (8, draft)):
                for bad in (False, True) if t > 1 else (False,):
                    q = torch.randn(2, t, hk * group, d, generator=gen).to(dtype).to(DEV)
                    fc.paged_cache_write_fp4(k, v, cache, slots)  # (and over the last one's scales of NaN)
                    if bad:
                        cache[2][first[(n - 1) // page].long(), (n - 1) % page] = 255
                        cache[3][first[(n - 2) // page].long(), (n - 2) % page, :, -1] = 255
                    print(f"[past 32 bits] {d} {dtype} rows {group * t} bad {bad}", flush=True)
                    o = fc.paged_decode_attention_fp4(q, cache, table, lengths, d ** -0.5, 60, 3)
                    assert torch.count_nonzero(o[1]) == 0
                    for i in range(t):
                        m = n - t + 1 + i
                        if bad and i == t - 1:
                            assert torch.isnan(o[0, i]).all()
                            continue
                        ref = oa.attention(f64(q[0, i:i + 1]), held_k[:m], held_v[:m], d ** -0.5, 60, 3, dtype=NAMES[dtype])
                        got, hidden = o[0, i:i + 1], d - 32 if bad and i == t - 2 else d
                        assert not torch.isfinite(got[..., hidden:]).any()
                        compare(f"token {i}", got[..., :hidden], ref["o"][..., :hidden], ref["o_tol"][..., :hidden])


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float16, 128)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("draft,hq", [(1, 2), (3, 16)])
def test_scores_at_the_ends_of_the_range(dtype, d, sign, draft, hq):
    """Equal scores near float32's ends, in one part and in parts that are joined: means of the values."""
    lengths = [40, 9000, 700]
    q, cache, table, lens = make(lengths, 16, hq, 2, d, draft, dtype, 39)
    q.zero_(), cache.k.zero_()
    q[..., 0] = 1.0
    cache.k[..., 0] = 0x06 if sign > 0 else 0x0e  # 4
    cache.k_scale.fill_(252)                      # 2^125
    for scale in (0.75, 4.0):
        o, lse = fc.paged_decode_attention_fp4(q, cache, table, lens, scale, return_lse=True)
        want = min(2.0 ** 127 * scale, torch.finfo(torch.float32).max) * sign
        assert torch.isfinite(lse).all() and (lse.double() - want).abs().max() <= 2 ** -7 * abs(want)
        for b, n in enumerate(lengths):
            v = rows(cache, table, b, n)[1]
            for t in range(draft):
                mean = v[:n - draft + 1 + t].mean(0).repeat(hq // 2, 0)
                u = max(oa.UNIT[NAMES[dtype]], n * 2.0 ** -24)
                assert (np.abs(f64(o[b, t]) - mean) <= 4 * u * np.abs(v).max()).all()


# ----------------------------------------------------------------------------
# Writing and reading back.
# ----------------------------------------------------------------------------
def hard_rows(n, heads, d, dtype, seed):
    """Rows over the type's whole range: ties, blocks of zeros, one value, infinities and NaN."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=gen)
    span = 12 if dtype == torch.float16 else 100
    x = x * 2.0 ** torch.randint(-span, span, (n, heads, 1), generator=gen)
    x[::5] = torch.randint(-14, 15, x[::5].shape, generator=gen) / 4.0  # halves of the steps
    x[1, :, :32] = 0
    x[2, :, 3] = torch.inf
    x[3, 0, 33] = torch.nan
    x[4 % n, :, :] = -0.0
    x = x.to(dtype)
    x[6 % n, :, 5], x[7 % n, 0, 7] = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    return x.to(DEV)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 256)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_write_and_read(dtype, d, heads_first):
    """Rows land where their slots say, rounded as defined; skipped slots and all other
    rows stay; contexts come back packed."""
    gen = torch.Generator().manual_seed(28)
    pages, page, hk, n = 9, 13, 3, 70
    cache = filled(pages, page, hk, d, 5, heads_first)
    kv = torch.cat([hard_rows(n, hk, d, dtype, s).flatten(1) for s in (1, 2)], 1)
    k, v = (x.view(n, hk, d) for x in kv.split(hk * d, -1))  # strided rows
    slots = torch.randperm(pages * page, generator=gen)[:n]
    slots[5], slots[17], slots[40] = -1, pages * page, 2 ** 40
    keep = (slots >= 0) & (slots < pages * page)
    want = [x.clone().reshape(pages * page, hk, -1) for x in cache]
    for i, x in enumerate((k, v)):
        data, scales = of.quantise(f64(x))
        want[i][slots[keep].to(DEV)] = torch.from_numpy(data).to(DEV)[keep.to(DEV)]
        want[2 + i][slots[keep].to(DEV)] = torch.from_numpy(scales).to(DEV)[keep.to(DEV)]
    versions = [x._version for x in cache]
    fc.paged_cache_write_fp4(k, v, cache, slots.to(DEV))
    assert all(x._version > a for x, a in zip(cache, versions))
    got = [x.reshape(pages * page, hk, -1) for x in cache]
    for i in range(2):
        assert torch.equal(got[2 + i], want[2 + i])
        # (codes of NaN's scale stand for nothing, and of zero there are two)
        a, b = held(got[i], got[2 + i]), held(want[i], want[2 + i])
        np.testing.assert_array_equal(a, b)
    table = torch.tensor([[3, 8, 1], [0, -1, 5], [2, 4, 100]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([30, 39, 28], dtype=torch.int32, device=DEV)
    for out in (torch.bfloat16, torch.float32, dtype):
        ks, vs, cu = fc.paged_cache_read_fp4(cache, table, lengths, 105, out)
        assert cu.tolist() == [0, 30, 69, 97] and ks.dtype == out and cu.dtype == torch.int32
        for i, x in enumerate((ks, vs)):
            flat = held(cache[i], cache[2 + i]).reshape(pages, page, hk, d)
            ref = np.zeros((105, hk, d))
            for b, (start, length) in enumerate(((0, 30), (30, 39), (69, 28))):
                for j in range(length):
                    g = int(table[b, j // page])
                    if 0 <= g < pages:
                        ref[start + j] = flat[g, j % page]
            if out == torch.float16:
                with np.errstate(over="ignore"):
                    ref = ref.astype(np.float16).astype(np.float64)
            np.testing.assert_array_equal(f64(x), ref)


def test_write_of_other_shapes():
    """Leading axes, int32 slots, rows 8 bytes off the alignment, v in another type."""
    hk, d = 2, 64
    gen = torch.Generator().manual_seed(7)
    cache = fc.fp4_cache(4, 8, hk, d, DEV)
    k, v = (torch.randn(2, 3, hk, d, generator=gen).to(DEV) for _ in range(2))
    fc.paged_cache_write_fp4(k, v.to(torch.bfloat16), cache, torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3))
    wide = torch.randn(10, hk * d + 8, generator=gen).to(torch.bfloat16).to(DEV)[:, 4:4 + hk * d].unflatten(-1, (hk, d))
    assert wide.data_ptr() % 16 == 8
    fc.paged_cache_write_fp4(wide, wide, cache, torch.arange(16, 26, device=DEV))
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    ks, vs, _ = fc.paged_cache_read_fp4(cache, table, torch.tensor([32], dtype=torch.int32, device=DEV), 32, torch.float32)
    for got, first in ((ks, k), (vs, v.to(torch.bfloat16))):
        ref = np.zeros((32, hk, d))
        ref[:6] = of.values(*of.quantise(f64(first).reshape(6, hk, d)))
        ref[16:26] = of.values(*of.quantise(f64(wide)))
        np.testing.assert_array_equal(f64(got), ref)
    empty = torch.zeros(0, hk, d, device=DEV)
    fc.paged_cache_write_fp4(empty, empty, cache, torch.zeros(0, dtype=torch.int64, device=DEV))


@pytest.mark.parametrize("batch", [1, 255, 257, 4096])
def test_read_of_many_sequences(batch):
    """Sequences of uneven lengths, none among them, cut where the rows end."""
    page, hk, d = 4, 1, 64
    lengths = [(i * 7) % 11 - 1 for i in range(batch)]
    cache = filled(64, page, hk, d, 9)
    gen = torch.Generator().manual_seed(11)
    table = torch.randint(64, (batch, 3), generator=gen).to(torch.int32).to(DEV)
    total = sum(max(n, 0) for n in lengths)
    for tokens in (total, max(0, total - 5), total + 9):
        k, v, cu = fc.paged_cache_read_fp4(cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), tokens,
                                           torch.float32)
        ref_cu = np.minimum(np.concatenate(([0], np.cumsum([max(n, 0) for n in lengths]))), tokens)
        np.testing.assert_array_equal(to_numpy(cu), ref_cu)
        for i, x in enumerate((k, v)):
            flat = held(cache[i], cache[2 + i])
            ref = np.zeros((total + 9, hk, d))
            at_ = 0
            for b, n in enumerate(lengths):
                for j in range(max(n, 0)):
                    ref[at_] = flat[int(table[b, j // page]), j % page] if batch <= 257 or b % 97 == 0 else np.nan
                    at_ += 1
            seen = ~np.isnan(ref[:tokens]).any((1, 2))
            np.testing.assert_array_equal(f64(x)[seen], ref[:tokens][seen])


def test_numbers_past_32_bits():
    """64-bit lengths and table entries that 32 bits do not hold: no such keys, no such pages."""
    q, cache, table, lengths = make([90, 40, 60], 16, 4, 2, 64, 1, torch.bfloat16, 41)
    far, lens = table.long(), lengths.long()
    far[0, 2] += 2**32
    lens[1] -= 2**32
    hole, none = table.clone(), lengths.clone()
    hole[0, 2], none[1] = -1, 0
    assert torch.equal(fc.paged_decode_attention_fp4(q, cache, far, lens, 0.125),
                       fc.paged_decode_attention_fp4(q, cache, hole, none, 0.125))
    for x, y in zip(fc.paged_cache_read_fp4(cache, far, lens, 150), fc.paged_cache_read_fp4(cache, hole, none, 150)):
        assert torch.equal(x, y)


def test_empty_reads():
    cache = filled(4, 8, 2, 64, 2)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    k, v, cu = fc.paged_cache_read_fp4(cache, none.view(0, 3), none, 7)
    assert torch.count_nonzero(k) == 0 and torch.count_nonzero(v) == 0 and cu.tolist() == [0]
    one = torch.tensor([5], dtype=torch.int32, device=DEV)
    k, v, cu = fc.paged_cache_read_fp4(cache, none.view(0, 3).new_zeros(1, 0), one, 5)
    assert torch.count_nonzero(k) == 0 and cu.tolist() == [0, 5]
    k, v, cu = fc.paged_cache_read_fp4(cache, one[None], one, 0)
    assert k.shape == (0, 2, 64) and cu.tolist() == [0, 0]


# ----------------------------------------------------------------------------
# As a program uses them.
# ----------------------------------------------------------------------------
def test_prompts_in_pieces_then_decoding():
    """A prompt's pieces attended over what the cache gives back, then tokens one at a time,
    against float64 attention over the whole rounded sequence."""
    torch.manual_seed(29)
    hq, hk, d, page, window, sinks, pieces = 8, 2, 64, 16, 60, 4, (70, 33, 50)
    n = sum(pieces) + 12
    q, k, v = (torch.randn(n, h, d, device=DEV).to(torch.bfloat16) for h in (hq, hk, hk))
    rounded = [of.values(*of.quantise(f64(x))) for x in (k, v)]
    ref = oa.attention(f64(q), *rounded, 0.125, window, sinks, dtype="bfloat16")
    cache = filled(20, page, hk, d, 1)
    cache.k_scale.fill_(255), cache.v_scale.fill_(255)
    table = torch.randperm(20, device=DEV).to(torch.int32)[None]
    slots = table[0].long().repeat_interleave(page) * page + torch.arange(20 * page, device=DEV) % page
    at_ = 0
    for m in pieces:
        fc.paged_cache_write_fp4(k[at_:at_ + m], v[at_:at_ + m], cache, slots[at_:at_ + m])
        at_ += m
        ks, vs, cu = fc.paged_cache_read_fp4(cache, table, torch.tensor([at_], dtype=torch.int32, device=DEV), at_)
        o = at.window_attention(q[None, at_ - m:at_], ks[None], vs[None], 0.125, window, sinks,
                                torch.tensor([0, m], dtype=torch.int32, device=DEV), cu)
        compare("piece", o[0], ref["o"][at_ - m:at_], ref["o_tol"][at_ - m:at_])
    for t in range(at_, n):
        fc.paged_cache_write_fp4(k[t:t + 1], v[t:t + 1], cache, slots[t:t + 1])
        o = fc.paged_decode_attention_fp4(q[None, t:t + 1], cache, table,
                                          torch.tensor([t + 1], dtype=torch.int32, device=DEV), 0.125, window, sinks)
        compare("token", o[0], ref["o"][t:t + 1], ref["o_tol"][t:t + 1])


def test_equal_runs_and_graph_replay():
    """Captured and replayed several times among eager work, each replay bit-equal."""
    q, cache, table, lengths = make([3000, 17, 900, 0], 16, 8, 2, 128, 1, torch.bfloat16, 27)
    k, v = (torch.randn(4, 2, 128, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([table[0, 2999 // 16].item() * 16 + 2999 % 16, -1, 10 ** 9, -7], device=DEV)

    def step():
        fc.paged_cache_write_fp4(k, v, cache, slots)
        return (fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.09, 500, 4),
                *fc.paged_cache_read_fp4(cache, table, lengths, 3920))

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
        for x in out:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(out, want, step()):
            assert torch.equal(x, y) and torch.equal(z, y)


def test_compiled_calls_equal_eager():
    q, cache, table, lengths = make([300, 17, 90], 16, 8, 2, 64, 1, torch.bfloat16, 32)
    k, v = (torch.randn(3, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = torch.stack([table[b, (n - 1) // 16] * 16 + (n - 1) % 16 for b, n in enumerate((300, 17, 90))]).long()

    def step(q, k, v, kc, vc, ks, vs, slots):
        cache = (kc, vc, ks, vs)
        fc.paged_cache_write_fp4(k, v, cache, slots)
        rows_k, rows_v, cu = fc.paged_cache_read_fp4(cache, table, lengths, 407, torch.float32)
        return fc.paged_decode_attention_fp4(q * 2, cache, table, lengths, 0.125, 50, 3) + 1, rows_k, rows_v, cu

    other = [x.clone() for x in cache]
    with torch.no_grad():
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, v, *other, slots)
        want = step(q, k, v, *cache, slots)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(other, cache))


def test_ops_pass_the_opcheck():
    q, cache, table, lengths = make([30, 7], 16, 4, 2, 64, 1, torch.float32, 33)
    k, v = (torch.randn(2, 2, 64, device=DEV) for _ in range(2))
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(fc.paged_decode_attention_fp4_op, (q, *cache, table, lengths, 0.125, 8, 1), test_utils=utils)
    torch.library.opcheck(fc.paged_cache_write_fp4_op, (k, v, *cache, torch.tensor([3, 20], device=DEV)), test_utils=utils)
    torch.library.opcheck(fc.paged_cache_read_fp4_op, (*cache, table, lengths, 40, torch.float32), test_utils=utils)


def test_side_stream_and_out():
    """A call on another stream than the current one's, into a given output."""
    q, cache, table, lengths = make([700, 90], 16, 4, 2, 64, 2, torch.bfloat16, 34)
    want, lse = fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.125, return_lse=True)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.125, out=out)
    side.synchronize()
    assert got is out and torch.equal(out, want)
    with pytest.raises(ValueError, match="out must"):
        fc.paged_decode_attention_fp4(q, cache, table, lengths, 0.125, out=out.float())


DEBUG = {
    "pages": lambda: test_pages_windows_and_lengths(7, 40, 5),
    "drafts": lambda: test_head_groups_and_drafts(24, 8, 4),
    "joined parts": test_long_contexts_are_split_and_joined,
    "float32, 256 wide": lambda: test_widths_and_types(256, torch.float32, False),
    "write and read": lambda: test_write_and_read(torch.bfloat16, 128, True),
    "many sequences": lambda: test_read_of_many_sequences(257),
}


@pytest.mark.parametrize("case", DEBUG)
def test_under_the_debug_build(case):
    """LDS, outputs and workspaces filled with NaN first."""
    with _lib.debug_library():
        DEBUG[case]()
