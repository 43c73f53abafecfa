"""The page pool on the device, number by number against the oracle (oracle/pages.py):
padding, refusals, pools that run out, many requests, steps in a captured graph."""
import random

import pytest
import torch

from oracle import pages as op
from pseudobrain_amd import _lib
from pseudobrain_amd import attention as at
from pseudobrain_amd import pages as pg

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def held_table(lengths, page, width, rng, extra):
    """Rows of distinct pages for these lengths, and `extra` more pages as the pool."""
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = list(range(sum(need) + extra))
    rng.shuffle(pages)
    rows = [[pages.pop() for _ in range(min(n, width))] + [-1] * (width - n) for n in need]
    return rows, pages[:extra]


def check_extend(lengths, counts, page, width, extra, tokens, seed, spare=5):
    rng = random.Random(seed)
    rows, pool = held_table(lengths, page, width, rng, extra)
    table, free = ints(rows).view(len(lengths), width), ints(pool + [-7] * spare)
    got = pg.paged_cache_extend(table, ints(lengths), ints(counts), free, ints([len(pool)]), page, tokens)
    again = pg.paged_cache_extend(table, ints(lengths), ints(counts), free, ints([len(pool)]), page, tokens)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    assert free.tolist() == pool + [-7] * spare
    want = op.extend(rows, lengths, counts, pool, page, tokens)
    slots, positions, cu, after, left = (x.tolist() for x in got)
    assert (slots, positions, cu, after, left) == (*want, [len(pool)])
    assert table.tolist() == rows
    assert got[0].dtype == torch.int64 and all(x.dtype == torch.int32 for x in got[1:])
    return want


@pytest.mark.parametrize("page", [1, 7, 16, 528])
@pytest.mark.parametrize("extra", [0, 3, 40, 2000])
def test_extend(page, extra):
    """Padding, requests at the ends of pages, prompts, pools of no page and enough."""
    lengths = [0, 5, page, page - 1, 2 * page, 0, 3 * page + 1, 100, 0]
    counts = [1, 1, 1, 1, 0, -3, 2, 300, 777]
    check_extend(lengths, counts, page, 1500, extra, 1200, page + extra)
    check_extend(lengths, counts, page, 1500, extra, 300, page + extra)   # the prompts' tokens do not fit
    check_extend(lengths, counts, page, max(5, 120 // page + 1), extra, 1200, page + extra)  # nor their rows


def test_refused_requests_leave_the_others_theirs():
    lengths, counts = [-1, 0, 16, 15, 8, 30], [4, 33, 1, 1, 8, 1]
    slots, positions, cu, after = check_extend(lengths, counts, 16, 4, 2, 100, 1)
    # no length; three pages of two; wants one past them; none needed; none; none
    assert after == [-1, 0, 16, 16, 16, 31] and cu == [0, 0, 0, 0, 1, 9, 10]


@pytest.mark.parametrize("batch", [1, 64, 255, 256, 257, 1000, 4096])
def test_many_requests(batch):
    rng = random.Random(batch)
    lengths = [rng.choice([0, 0, 3, 16, 31, 64, 77]) for _ in range(batch)]
    counts = [rng.choice([0, 1, 1, 5, 40]) for _ in range(batch)]
    check_extend(lengths, counts, 16, 9, batch // 2, sum(counts), batch)
    check_extend(lengths, counts, 16, 9, 3 * batch, sum(counts) * 2 // 3, batch)


def test_counts_that_would_overflow():
    big = 2 ** 31 - 1
    check_extend([5, 0, 7, 9], [big, big, big, 2], 16, 4, 9, 100, 2)
    check_extend([5, 7, 0], [1, 2, big], 16, 4, 9, 100, 2)


@pytest.mark.parametrize("page", [1, 4, 16])
def test_release(page):
    rng = random.Random(page)
    width, batch = 40, 70
    rows = [[rng.randrange(10 ** 6) for _ in range(width)] for _ in range(batch)]
    first = [rng.choice([0, 0, 1, page, 3 * page - 1, 17, -5]) for _ in range(batch)]
    end = [max(0, a) + rng.choice([0, 1, page - 1, page, 5 * page + 3, 10 ** 6, -9]) for a in first]
    for start, spare in ((0, 5000), (13, 5000), (13, 100), (3, 0)):
        pool = [rng.randrange(10 ** 6) for _ in range(start)]
        free = ints(pool + [-7] * spare)
        left = pg.paged_cache_release(ints(rows), ints(first), ints(end), free, ints([start]), page)
        capacity = start + spare
        op.release(rows, [max(0, a) for a in first], end, pool, page, capacity)
        assert left.tolist() == [len(pool)]
        assert free.tolist() == pool + [-7] * (capacity - len(pool))


@pytest.mark.parametrize("batch,width", [(1, 3), (7, 40), (1, 70000), (5, 9000), (300, 500), (4096, 6)])
@pytest.mark.parametrize("absent", [0.0, 0.3, 1.0])
def test_absent_entries_do_not_come_back_as_pages(batch, width, absent):
    """Ranges with entries below 0 among them, in one workgroup's run and over many, pools with room for
    all and for some."""
    page, rng = 4, random.Random(batch + width)
    gen = torch.Generator().manual_seed(batch)
    rows = torch.randint(10 ** 6, (batch, width), generator=gen)
    rows[torch.rand(batch, width, generator=gen) < absent] = -1
    rows = rows.tolist()
    first = [rng.choice([0, 0, 0, 5, page * width]) for _ in range(batch)]
    end = [rng.choice([page * width, page * width, 10 ** 9, page * (width // 2) + 1, 0]) for _ in first]
    first[0], end[0] = 0, page * width
    for start, spare in ((3, batch * width), (3, batch * width // 3), (0, 0)):
        pool = list(range(start))
        free = ints(pool + [-7] * spare)
        left = pg.paged_cache_release(ints(rows), ints(first), ints(end), free, ints([start]), page)
        op.release(rows, first, end, pool, page, start + spare)
        assert left.tolist() == [len(pool)]
        assert free.tolist() == pool + [-7] * (start + spare - len(pool))


def test_a_pool_over_absent_entries_grants_pages():
    """A request that held its window's pages alone gives them back; what the pool then grants is pages."""
    table, free = ints([[-1, -1, 5, -1, 6]]), ints([9, -7, -7, -7])
    num_free = pg.paged_cache_release(table, ints([0]), ints([20]), free, ints([1]), 4)
    assert num_free.tolist() == [3] and free.tolist() == [9, 5, 6, -7]
    slots, *_, left = pg.paged_cache_extend(table, ints([0]), ints([20]), free, num_free, 4, 20)
    assert left.tolist() == [3] and slots.tolist() == [-1] * 20  # five pages are not there
    slots, *_, left = pg.paged_cache_extend(table, ints([0]), ints([12]), free, num_free, 4, 12)
    assert left.tolist() == [0] and slots.tolist() == [*range(24, 28), *range(20, 24), *range(36, 40)]


def test_numbers_past_32_bits():
    """64-bit lengths, counts and ranges that 32 bits do not hold."""
    far = torch.iinfo(torch.int64).max
    free = ints([0, 0, 0, 0])
    left = pg.paged_cache_release(ints([[4, 5], [6, 7]]), ints([0, far], torch.int64), ints([far, far], torch.int64), free,
                                  ints([1], torch.int64), 16)
    assert left.tolist() == [3] and free.tolist() == [0, 4, 5, 0]
    slots, _, cu, after, left = pg.paged_cache_extend(
        ints([[-1, -1]] * 4), ints([0, 2**32, 5 - 2**32, 0], torch.int64), ints([3, 1, 1, 2**32 + 1], torch.int64),
        ints([8, 9]), ints([2**32 + 1], torch.int64), 16, 9)
    assert cu.tolist() == [0, 3, 3, 3, 3] and slots.tolist() == [144, 145, 146] + [-1] * 6
    assert after.tolist() == [3, 2**31 - 1, -2**31, 0] and left.tolist() == [1]


def test_empty_calls_and_strided_tables():
    none = ints([])
    slots, positions, cu, after, left = pg.paged_cache_extend(none.view(0, 3), none, none, ints([4, 5]), ints([2]), 16, 6)
    assert slots.tolist() == positions.tolist() == [-1] * 6 and cu.tolist() == [0] and left.tolist() == [2]
    out = pg.paged_cache_extend(ints([[0]]), ints([0]), ints([1]), none, ints([0]), 16, 0)
    assert out[0].numel() == 0 and out[2].tolist() == [0, 0] and out[3].tolist() == [0] and out[4].tolist() == [0]
    assert pg.paged_cache_release(none.view(0, 3), none, none, none, ints([0]), 16).tolist() == [0]
    wide = ints([[-1] * 7, [-1] * 7])
    slots, *_ = pg.paged_cache_extend(wide[:, 2:5], ints([0, 0], torch.int64), ints([17, 3], torch.int64), ints([4, 8, 6]),
                                      ints([3], torch.int64), 16, 20)
    assert wide.tolist() == [[-1, -1, 6, 8, -1, -1, -1], [-1, -1, 4, -1, -1, -1, -1]]
    assert slots.tolist() == [*range(96, 112), 128, 64, 65, 66]
    # a pool's height beyond its capacity, or below nothing
    assert pg.paged_cache_extend(ints([[-1]]), ints([0]), ints([1]), ints([9]), ints([55]), 16, 1)[4].tolist() == [0]
    assert pg.paged_cache_extend(ints([[-1]]), ints([0]), ints([1]), ints([9]), ints([-2]), 16, 1)[3].tolist() == [0]


def test_steps_in_a_captured_graph():
    """Requests growing by what the device decides, their windows' pages given back, step
    after step by replays of one graph, against the oracle."""
    page, batch, width, window, capacity = 4, 5, 40, 10, 24
    rng = random.Random(3)
    rows, pool = [[-1] * width for _ in range(batch)], list(range(capacity))
    rng.shuffle(pool)
    table, free = ints(rows), ints(pool)
    lengths, low, num_free = ints([0] * batch), ints([0] * batch), ints([capacity])
    counts = ints([0] * batch)
    out = [torch.zeros(12, dtype=d, device=DEV) for d in (torch.int64, torch.int32)]

    def step():
        after = (lengths - window).clamp(min=0)
        num_free.copy_(pg.paged_cache_release(table, low, after, free, num_free, page))
        low.copy_(after)
        slots, positions, _, new, left = pg.paged_cache_extend(table, lengths, counts, free, num_free, page, 12)
        for x, y in ((lengths, new), (num_free, left), (out[0], slots), (out[1], positions)):
            x.copy_(y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (no counts: nothing moves)
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    n, lo = [0] * batch, [0] * batch
    for i in range(40):
        c = [rng.choice([0, 1, 2, 4]) for _ in range(batch)]
        counts.copy_(torch.tensor(c))
        graph.replay()
        torch.cuda.synchronize()
        after = [max(0, x - window) for x in n]
        op.release(rows, lo, after, pool, page, capacity)
        lo = after
        slots, positions, _, n = op.extend(rows, n, c, pool, page, 12)
        assert out[0].tolist() == slots and out[1].tolist() == positions
        assert lengths.tolist() == n and num_free.tolist() == [len(pool)] and free.tolist()[:len(pool)] == pool
        assert table.tolist() == rows


def test_slots_reach_the_cache():
    """Tokens written at the slots are found by the page table."""
    torch.manual_seed(1)
    page, hk, d = 16, 2, 64
    kc, vc = (torch.zeros(12, page, hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table, free = ints([[-1] * 5] * 3), ints(torch.randperm(12).tolist())
    lengths, num_free = ints([0, 0, 0]), ints([12])
    k = torch.randn(80, hk, d, device=DEV).to(torch.bfloat16)
    seen = [[], [], []]
    for counts in ([20, 0, 33], [1, 1, 1], [15, 4, 1]):
        slots, positions, cu, lengths, num_free = pg.paged_cache_extend(table, lengths, ints(counts), free, num_free, page, 80)
        at.paged_cache_write(k, k, kc, vc, slots)
        for b in range(3):
            seen[b] += k[cu[b]:cu[b + 1]].unbind(0)
    for b in range(3):
        n = lengths[b].item()
        assert n == len(seen[b])
        rows = kc[table[b, :-(-n // page)].long()].flatten(0, 1)[:n]
        assert torch.equal(rows, torch.stack(seen[b]))


def test_versions_compilation_and_the_opcheck():
    def args():
        return ints([[3, -1, -1], [5, 6, -1]]), ints([16, 20]), ints([3, 1]), ints([1, 2, 4]), ints([3])

    a = args()
    versions = a[0]._version, a[3]._version
    pg.paged_cache_extend(*a, 16, 8)
    assert a[0]._version > versions[0] and a[3]._version == versions[1]
    pg.paged_cache_release(a[0], ints([0, 0]), ints([16, 16]), a[3], ints([0]), 16)
    assert a[3]._version > versions[1]

    def both(table, lengths, counts, free, num_free):
        out = pg.paged_cache_extend(table, lengths, counts, free, num_free, 16, 8)
        return (*out, pg.paged_cache_release(table, lengths * 0, lengths, free, out[4], 16))

    x, y = args(), args()
    want, got = both(*x), torch.compile(both, backend="aot_eager", fullgraph=True)(*y)
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and all(torch.equal(p, q) for p, q in zip(x, y))
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(pg.paged_cache_extend_op, (*args(), 16, 8), test_utils=utils)
    table, lengths, _, free, num_free = args()
    torch.library.opcheck(pg.paged_cache_release_op, (table, lengths * 0, lengths, free, num_free * 0, 16), test_utils=utils)


@pytest.mark.parametrize("case", ["extend", "release", "many"])
def test_under_the_debug_build(case):
    with _lib.debug_library():
        dict(extend=lambda: test_extend(16, 40), release=lambda: test_release(4), many=lambda: test_many_requests(1000))[case]()
