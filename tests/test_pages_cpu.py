"""The page pool without a GPU: the oracle against what must hold of any pool, the C
ABI's and the host API's refusals."""
import random

import pytest
import torch

from oracle import pages as op
from pseudobrain_amd import _lib
from pseudobrain_amd import pages as pg
from tests.test_attention_cpu import FAKE


def test_no_page_is_held_twice_or_lost():
    """Requests that grow, slide their windows and end, in turn with a pool too small for all."""
    rng = random.Random(0)
    page, batch, width, capacity = 4, 6, 20, 30
    pool, table = list(range(capacity)), [[-1] * width for _ in range(batch)]
    lengths, given = [0] * batch, [0] * batch
    refused = 0
    for _ in range(400):
        counts = [rng.choice([0, 1, 1, 7]) for _ in range(batch)]
        before = lengths
        slots, positions, cu, lengths = op.extend(table, lengths, counts, pool, page, 20)
        refused += sum(n == m and c > 0 for n, m, c in zip(before, lengths, counts))
        held = [table[b][i] for b in range(batch) for i in range(given[b] // page, -(-lengths[b] // page))]
        assert len(set(held + pool)) == len(held) + len(pool) == capacity
        live = [s for s in slots if s >= 0]
        assert len(set(live)) == len(live) == cu[-1]
        for b in range(batch):
            for t in range(cu[b], cu[b + 1]):
                assert slots[t] == table[b][positions[t] // page] * page + positions[t] % page
        first = list(given)
        for b in range(batch):
            if rng.random() < 0.1 or lengths[b] > 60:
                given[b] = -(-lengths[b] // page) * page  # a finished request
            else:
                given[b] = max(given[b], (lengths[b] - 24))
        op.release(table, first, given, pool, page, capacity)
        for b in range(batch):
            if given[b] >= lengths[b] and lengths[b] % page == 0 or given[b] > lengths[b]:
                lengths[b] = given[b] = 0
    assert refused > 50


@pytest.mark.parametrize("released", [True, False])
def test_drafts_that_are_not_accepted(released):
    """Lengths that go back: with the pages between released first none is lost, without they are."""
    rng = random.Random(1)
    page, batch, width, capacity, draft = 4, 3, 40, 40, 6
    pool, table = list(range(capacity)), [[-1] * width for _ in range(batch)]
    lengths = [0] * batch
    for _ in range(30):
        before = lengths
        *_, lengths = op.extend(table, lengths, [draft] * batch, pool, page, draft * batch)
        accepted = [min(n, m + rng.randint(0, draft)) for n, m in zip(lengths, before)]
        if released:
            up = [[-(-n // page) * page for n in x] for x in (accepted, lengths)]
            op.release(table, *up, pool, page, capacity)
        lengths = accepted
        held = [row[i] for row, n in zip(table, lengths) for i in range(-(-n // page))]
        assert len(set(held + pool)) == len(held) + len(pool)
        assert not released or len(held) + len(pool) == capacity
    assert min(lengths) > 5 * page and (released or len(held) + len(pool) < capacity)


def test_absent_entries_are_not_released():
    pool = [7]
    op.release([[3, -1, 4], [-1, -1, -1]], [0, 0], [12, 12], pool, 4, 9)
    assert pool == [7, 3, 4]


def extend(**over):
    args = dict(table=FAKE, row=4, max_pages=4, lengths=FAKE, counts=FAKE, B=2, page=16, free=FAKE, capacity=9,
                num_free=FAKE, tokens=3, slots=FAKE, positions=FAKE, cu=FAKE, after=FAKE, left=FAKE, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_pages_extend(*args.values())


def release(**over):
    args = dict(table=FAKE, row=4, max_pages=4, first=FAKE, end=FAKE, B=2, page=16, free=FAKE, capacity=9, num_free=FAKE,
                left=FAKE, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_pages_release(*args.values())


POOL = [
    (dict(B=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(B=pg.MAX_REQUESTS + 1), _lib.ERR_UNSUPPORTED),
    (dict(max_pages=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(page=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(page=1 << 20, max_pages=1 << 11), _lib.ERR_UNSUPPORTED),  # 2^31 tokens
    (dict(row=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(capacity=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(table=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(free=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(num_free=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(left=None), _lib.ERR_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("over,code", POOL + [
    (dict(tokens=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(lengths=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(counts=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(slots=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(positions=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(cu=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(after=None), _lib.ERR_INVALID_ARGUMENT),
])
def test_extend_rejects(over, code):
    assert extend(**over) == code


@pytest.mark.parametrize("over,code", POOL + [
    (dict(first=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(end=None), _lib.ERR_INVALID_ARGUMENT),
])
def test_release_rejects(over, code):
    assert release(**over) == code


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_calls_refuse(monkeypatch):
    with pytest.raises(RuntimeError, match="no CPU path"):
        pg.paged_cache_extend(ints(2, 4), ints(2), ints(2), ints(9), ints(1), 16, 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pg.paged_cache_release(ints(2, 4), ints(2), ints(2), ints(9), ints(1), 16)
    monkeypatch.setattr(pg, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(pg, "_launch", lambda *args: pytest.fail("launched"))
    good = dict(table=ints(2, 4), a=ints(2), b=ints(2), free=ints(9), num=ints(1), page=16)
    many = pg.MAX_REQUESTS + 1
    for over, message in (
            (dict(a=ints(3)), "for each of its B requests"), (dict(b=ints(2, 1)), "for each"), (dict(table=ints(8)), "for each"),
            (dict(num=ints(2)), "num_free"), (dict(free=ints(3, 3)), "free_pages"), (dict(table=ints(2, 4).long()), "int32"),
            (dict(free=ints(9).long()), "int32"), (dict(table=ints(2, 8)[:, ::2]), "dense"),
            (dict(table=ints(1, 4).expand(2, 4)), "dense"), (dict(free=ints(18)[::2]), "dense"), (dict(page=0), "at least one"),
            (dict(page=2 ** 29), "2\\^31"), (dict(table=ints(many, 1), a=ints(many), b=ints(many)), "at most")):
        args = list({**good, **over}.values())
        with pytest.raises(ValueError, match=message):
            pg.paged_cache_release(*args)
        with pytest.raises(ValueError, match=message):
            pg.paged_cache_extend(*args, 3)
    with pytest.raises(ValueError, match="tokens"):
        pg.paged_cache_extend(*good.values(), -1)
    i32 = torch.int32
    with pytest.raises(ValueError, match="free_pages"):  # (a pool that a 32-bit count calls empty)
        pg._pool_plan((2, 4), (4, 1), (i32, i32), (2,), (2,), (2**32,), (1,), (1,), 16)
