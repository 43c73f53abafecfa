"""The operators around the attention's cache together, as a serving engine uses them:
pages and slots from the requests' lengths, norms and rotation by the positions that come
with them, writes into the 4-bit cache, prompts attended over what it gives back and
tokens decoded over it, pages given back behind the window and by finished requests."""
import numpy as np
import pytest
import torch

from oracle import attention as oa
from oracle import fp4 as of
from oracle import rope as orp
from pseudobrain_amd import (fp4_cache, paged_cache_extend, paged_cache_read_fp4, paged_cache_release,
                             paged_cache_write_fp4, paged_decode_attention_fp4, qk_norm_rope, rope_tables, window_attention)
from tests.test_gpu_window_attention import compare, f64

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HK, D, R, PAGE, WINDOW, SINKS, EPS = 8, 2, 64, 32, 16, 60, 4, 1e-6
KEPT = -(-SINKS // PAGE) * PAGE  # tokens whose pages the window never gives back
SCALE = D ** -0.5


class Engine:
    """Requests in fixed rows of a page table over one pool and one cache; what they have
    seen is kept on the host too, for the oracle."""

    def __init__(self, rows, pages, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.gen, self.rows = gen, rows
        self.cache = fp4_cache(pages, PAGE, HK, D, DEV)
        for scales in self.cache[2:]:
            scales.fill_(255)  # (what no request has written is NaN)
        self.table = torch.full((rows, 40), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
        self.num_free = torch.tensor([pages], dtype=torch.int32, device=DEV)
        self.lengths, self.low = (torch.zeros(rows, dtype=torch.int32, device=DEV) for _ in range(2))
        self.low.fill_(KEPT)
        self.weights = [(1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(torch.bfloat16) for _ in "qk"]
        self.cos, self.sin = rope_tables(1000, R, device=DEV)
        self.seen = [([], []) for _ in range(rows)]  # rounded keys and values of each request

    def tokens(self, n):
        """A projection's output for n tokens: q, k, v as columns of it."""
        x = torch.randn(1, n, (HQ + 2 * HK) * D, generator=self.gen, device=DEV).to(torch.bfloat16)
        return [y.unflatten(-1, (-1, D)) for y in x.split([HQ * D, HK * D, HK * D], -1)]

    def place(self, counts, tokens):
        """Behind the window, then the step's new tokens."""
        low = (self.lengths - WINDOW).clamp(min=KEPT)
        self.num_free = paged_cache_release(self.table, self.low, low, self.free, self.num_free, PAGE)
        self.low = low
        slots, positions, cu, self.lengths, self.num_free = paged_cache_extend(
            self.table, self.lengths, counts, self.free, self.num_free, PAGE, tokens)
        return slots, positions, cu

    def normed(self, q, k, positions):
        return qk_norm_rope(q, k, *self.weights, self.cos, self.sin, positions, EPS)

    def note(self, k, v, cu):
        """What the cache holds of the tokens written, and the normed rows against the oracle."""
        k, v = (of.values(*of.quantise(f64(x[0]))) for x in (k, v))
        for b in range(self.rows):
            for t in range(cu[b], cu[b + 1]):
                self.seen[b][0].append(k[t])
                self.seen[b][1].append(v[t])

    def check_normed(self, raw, got, positions):
        for x, y, w in zip(raw, got, self.weights):
            ref = orp.rows(f64(x), f64(w), f64(self.cos), f64(self.sin), positions.cpu().numpy()[None].astype(np.int64), EPS,
                           False, "bfloat16")
            compare("normed", y, ref["y"], ref["y_tol"])

    def expect(self, b, q):
        """The float64 attention of request b's newest len(q) tokens."""
        k, v = (np.stack(x) for x in self.seen[b])
        return oa.attention(q, k, v, SCALE, WINDOW, SINKS, dtype="bfloat16")

    def prefill(self, counts):
        tokens = sum(counts) + 5  # (padding: slots and positions of -1)
        slots, positions, cu = self.place(torch.tensor(counts, device=DEV, dtype=torch.int32), tokens)
        q, k, v = self.tokens(tokens)
        qr, kr = self.normed(q, k, positions)
        paged_cache_write_fp4(kr[0], v[0], self.cache, slots)
        total = int(self.lengths.sum())
        ks, vs, cu_k = paged_cache_read_fp4(self.cache, self.table, self.lengths, total + 3)
        o = window_attention(qr, ks[None], vs[None], SCALE, WINDOW, SINKS, cu, cu_k)
        self.check_normed((q, k), (qr, kr), positions)
        bounds = cu.tolist()
        self.note(kr, v, bounds)
        for b in range(self.rows):
            if bounds[b + 1] > bounds[b]:
                rows = slice(bounds[b], bounds[b + 1])
                ref = self.expect(b, f64(qr[0, rows]))
                compare(f"prompt {b}", o[0, rows], ref["o"], ref["o_tol"])
        assert torch.count_nonzero(o[0, bounds[-1]:]) == 0

    def decode(self, counts):
        """One token for the requests with counts of 1; the others' rows are padding."""
        counts_ = torch.tensor(counts, device=DEV, dtype=torch.int32)
        slots, positions, cu = self.place(counts_, self.rows)
        q, k, v = self.tokens(self.rows)
        qr, kr = self.normed(q, k, positions)
        paged_cache_write_fp4(kr[0], v[0], self.cache, slots)
        live = [b for b in range(self.rows) if counts[b]]
        qb = torch.zeros(self.rows, 1, HQ, D, dtype=torch.bfloat16, device=DEV)
        qb[live, 0] = qr[0, :len(live)]
        o = paged_decode_attention_fp4(qb, self.cache, self.table, self.lengths * counts_, SCALE, WINDOW, SINKS)
        self.note(kr, v, cu.tolist())
        for b in range(self.rows):
            if not counts[b]:
                assert torch.count_nonzero(o[b]) == 0
                continue
            ref = self.expect(b, f64(qb[b]))
            compare(f"token of {b}", o[b], ref["o"], ref["o_tol"])

    def finish(self, b):
        """All the request's pages back: the sinks', and those the window has not left."""
        mine = torch.arange(self.rows, device=DEV) == b
        zero = torch.zeros_like(self.lengths)
        rounded = (self.lengths + PAGE - 1) // PAGE * PAGE
        kept = rounded.clamp(max=KEPT)
        for first, end in ((zero, kept), (self.low, rounded)):
            self.num_free = paged_cache_release(self.table, first, torch.where(mine, end, zero).to(torch.int32), self.free,
                                                self.num_free, PAGE)
        self.lengths = torch.where(mine, zero, self.lengths)
        self.low = torch.where(mine, torch.full_like(zero, KEPT), self.low)
        self.seen[b] = ([], [])


def test_requests_come_and_go():
    pages = 34
    engine = Engine(4, pages, 1)
    engine.prefill([70, 0, 33, 1])
    engine.prefill([45, 100, 0, 17])  # two prompts' next pieces, and another request
    for _ in range(5):
        engine.decode([1, 1, 1, 1])
    engine.decode([1, 0, 0, 1])
    engine.finish(1)
    engine.prefill([0, 120, 0, 0])    # a new request in its row, over pages that others have left
    for _ in range(20):
        engine.decode([0, 1, 1, 1])
    for b in range(4):
        engine.finish(b)
    assert engine.num_free.item() == pages and sorted(engine.free.tolist()) == list(range(pages))


def test_drafts_partly_accepted():
    """Four drafted tokens a step, of which the device accepts some: rejected tokens' pages go back
    before the next step, their rows are written again, and no page is lost."""
    rows, pages, draft, steps = 3, 30, 4, 25
    engine = Engine(rows, pages, 4)
    engine.prefill([30, 1, 16])
    counts = torch.full((rows,), draft, dtype=torch.int32, device=DEV)

    def up(n):
        return (n + PAGE - 1) // PAGE * PAGE

    for i in range(steps):
        slots, positions, cu = engine.place(counts, rows * draft)
        assert cu.tolist() == [0, 4, 8, 12]
        q, k, v = engine.tokens(rows * draft)
        qr, kr = engine.normed(q, k, positions)
        paged_cache_write_fp4(kr[0], v[0], engine.cache, slots)
        o = paged_decode_attention_fp4(qr.view(rows, draft, HQ, D), engine.cache, engine.table, engine.lengths, SCALE,
                                       WINDOW, SINKS)
        engine.note(kr, v, cu.tolist())
        for b in range(rows):
            ref = engine.expect(b, f64(qr[0, draft * b:draft * (b + 1)]))
            compare(f"step {i}, drafts of {b}", o[b], ref["o"], ref["o_tol"])
        rejected = torch.randint(0, draft + 1, (rows,), generator=engine.gen, device=DEV)
        accepted = (engine.lengths - rejected).to(torch.int32)
        engine.num_free = paged_cache_release(engine.table, up(accepted), up(engine.lengths), engine.free, engine.num_free,
                                              PAGE)
        for b, n in enumerate(rejected.tolist()):
            for seen in engine.seen[b]:
                del seen[len(seen) - n:]
        engine.lengths = accepted
        held = [engine.table[b, j].item() for b in range(rows)
                for j in [*range(min(KEPT, up(accepted[b].item())) // PAGE),
                          *range(engine.low[b].item() // PAGE, up(accepted[b].item()) // PAGE)]]
        free = engine.free[:engine.num_free.item()].tolist()
        assert sorted(held + free) == list(range(pages))
    for b in range(rows):
        engine.finish(b)
    assert engine.num_free.item() == pages and sorted(engine.free.tolist()) == list(range(pages))


def test_a_pool_that_is_too_small():
    """What does not fit waits, and neither the others nor the pool notice."""
    engine = Engine(3, 6, 2)
    engine.prefill([40, 0, 0])  # three pages
    before = engine.lengths
    slots, positions, cu = engine.place(torch.tensor([1, 80, 30], dtype=torch.int32, device=DEV), 111)
    # (a request's wish counts before those after it, granted or not)
    assert engine.lengths.tolist() == [41, 0, 0] and cu.tolist() == [0, 1, 1, 1]
    assert (slots[1:] == -1).all() and (positions[1:] == -1).all() and before[0] == 40
    assert engine.num_free.item() == 3


def test_decode_steps_in_a_captured_graph():
    """Ten steps by replays of one graph, each against the same step taken eagerly."""
    rows, steps = 5, 10

    def start():
        engine = Engine(rows, 40, 3)
        engine.prefill([30, 7, 64, 16, 31])
        return engine

    x = torch.randn(steps, 1, rows, (HQ + 2 * HK) * D, device=DEV).to(torch.bfloat16)
    counts = torch.tensor([1, 1, 1, 0, 1], dtype=torch.int32, device=DEV)

    def step(engine, x):
        slots, positions, cu = engine.place(counts, rows)
        q, k, v = (y.unflatten(-1, (-1, D)) for y in x.split([HQ * D, HK * D, HK * D], -1))
        q, k = engine.normed(q, k, positions)
        paged_cache_write_fp4(k[0], v[0], engine.cache, slots)
        row = (torch.cumsum(counts, 0) - counts).clamp(max=rows - 1)
        return paged_decode_attention_fp4(q[0, row][:, None], engine.cache, engine.table, engine.lengths * counts, SCALE, WINDOW,
                                          SINKS)

    eager = start()
    want = [step(eager, x[i]) for i in range(steps)]
    engine, held = start(), torch.zeros_like(x[0])
    state = {n: getattr(engine, n).clone() for n in ("lengths", "low", "num_free")}

    def replayed():
        for n, t in state.items():
            setattr(engine, n, t)
        out = step(engine, held)
        for n, t in state.items():
            t.copy_(getattr(engine, n))
        return out

    saved = {n: t.clone() for n, t in state.items()}, engine.table.clone(), engine.free.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        replayed()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = replayed()
    for n, t in state.items():
        t.copy_(saved[0][n])
    engine.table.copy_(saved[1])
    engine.free.copy_(saved[2])
    for i in range(steps):
        held.copy_(x[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.count_nonzero(x[i]) > 0
    for n, t in state.items():
        assert torch.equal(t, getattr(eager, n))
