"""The workloads by which the speed of the operators around the attention's cache
is judged: what happens to a token's query and key before they are attended, where
a serving engine's tokens go, and the cache held in 4 bits.

Five kinds of call:

  rope    qk_norm_rope without gradients: the queries' and keys' norms of each
          head and their rotation
  train   qk_norm_rope and its backward through autograd
  pages   paged_cache_release and paged_cache_extend: pages that the window has
          left go back to the pool, the step's new tokens get pages and slots
  append  paged_cache_write_fp4 and paged_cache_read_fp4: a prompt's next piece
          into the 4-bit cache, and the whole context back for the attention
  decode  paged_decode_attention_fp4: the newest tokens of each running request
          against the 4-bit cache

The 4-bit cache. 32 consecutive values x of a head share a scale s, a power of two;
a value is held as the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} s (ties to the even
code). s = 2^(e - 2), 2^e being the largest |x| rounded to a power of two by its
first two mantissa bits (7 s and more would round to 8 s: the scale is doubled
there), held as the byte e - 2 + 127 within [2, 252]; 255 marks 32 values among
which one is infinite or NaN. Byte i of a head's row holds values 2 i (low half) and
2 i + 1.

The pages. Page i of a sequence holds its tokens i page .. i page + page - 1. Release
gives back, sequence by sequence, the pages whose last token lies in [first, end):
they are pushed on the stack free_pages, whose height is num_free. Extend goes through
the requests in order. One is granted if its tokens end within `tokens` (those of all
requests before it counted), its pages fit its row of the table, and the pages wanted
up to it do not exceed the pool's (or it wants none); it takes its pages from the top
of the stack. The tokens of the granted are packed: slot (page number times page size
plus place) and position of each, -1 past the last.

A case is a dict of plain values:
  kind, dtype, hq, hk, d
  rotary, interleaved, batch, length or seqs, tokens   (rope, train)
  batch, page, length, window, sinks, new, spare   (pages: longest context, most new tokens a
                                                    request, pages in the pool for each 100 wanted)
  seqs, tokens, cached, page, heads_first   (append: new tokens of all, longest context before)
  batch, length, page, draft, window, sinks, heads_first   (decode)
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
WIDE = dict(hq=32, hk=8, d=128)    # grouped heads of the usual width
K256 = dict(hq=16, hk=2, d=256)    # the widest heads, eight queries to a key head
SMALL = dict(hq=4, hk=4, d=64)     # the small float32 model: a key head for each query head
POSITIONS = 262144                 # rows of the rotation's tables
EPS = 1e-6
BLOCK = 32                         # values that share a scale
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(kind, dtype="bfloat16", heads=None, **sizes):
    return dict(kind=kind, dtype=dtype, **(WIDE if heads is None else heads), **sizes)


def listed():
    return [
        # a decode step: the newest token of 64 requests at far positions, a quarter of each wide head rotated
        dict(_case("rope", heads=K256, rotary=64, interleaved=False, batch=64, length=1), name="rope_b64"),
        # a serving engine's prefill batch of uneven prompts
        dict(_case("rope", rotary=128, interleaved=False, seqs=24, tokens=19001), name="rope_24seq_19001"),
        # a training batch
        dict(_case("train", rotary=128, interleaved=False, batch=4, length=2048), name="rope_train_4x2048"),
        # the small model's training step in float32, neighbouring values rotated
        dict(_case("train", dtype="float32", heads=SMALL, rotary=64, interleaved=True, batch=1, length=2048),
             name="rope_train_small_fp32"),
        # a decode step of a steady serving batch: a token each, small pages
        dict(_case("pages", batch=64, page=16, length=16384, window=4096, sinks=4, new=1, spare=100), name="pages_b64"),
        # a step that mixes prompts and running requests, an odd number of them, more pages wanted than there are
        dict(_case("pages", batch=233, page=16, length=8192, window=1024, sinks=64, new=160, spare=95),
             name="pages_b233_short"),
        # one user's short message onto a running conversation
        dict(_case("append", seqs=1, tokens=64, cached=256, page=16, heads_first=True), name="append_fp4_64"),
        # a prefill batch's next pieces, widest heads, large pages of no round size
        dict(_case("append", heads=K256, seqs=24, tokens=19001, cached=2000, page=528, heads_first=False),
             name="append_fp4_k256_19001"),
        # one user at the keyboard: latency only
        dict(_case("decode", batch=1, length=4097, page=16, draft=1, window=0, sinks=0, heads_first=True),
             name="decode_fp4_b1_4097"),
        # a steady serving batch of uneven contexts without a window
        dict(_case("decode", batch=64, length=16384, page=16, draft=1, window=0, sinks=0, heads_first=True),
             name="decode_fp4_b64_16384"),
        # a full serving batch of an odd size: window and sinks, four tokens to verify
        dict(_case("decode", heads=K256, batch=233, length=8192, page=528, draft=4, window=4096, sinks=64,
                   heads_first=False), name="decode_fp4_k256_b233_w4096"),
        # the small model in float32
        dict(_case("decode", dtype="float32", heads=SMALL, batch=24, length=2048, page=32, draft=1, window=0, sinks=0,
                   heads_first=False), name="decode_fp4_small_fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed kinds' ranges, none dearer than the dearest listed."""
    kind = rng.choice(["rope", "rope", "train", "pages", "append", "decode", "decode", "decode"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    heads = rng.choice([WIDE, K256, SMALL, dict(hq=24, hk=8, d=64), dict(hq=16, hk=16, d=128), dict(hq=14, hk=2, d=128)])
    page = rng.choice([16, 32, 64, 100, 528])
    first = rng.random() < 0.5
    if kind in ("rope", "train"):
        rotary = rng.choice([heads["d"], heads["d"] // 2, heads["d"] // 4])
        sizes = dict(rotary=rotary, interleaved=rng.random() < 0.3)
        tokens = _log_int(rng, 1, 19001 if kind == "rope" else 8192)
        many = _log_int(rng, 1, min(64, max(1, tokens // 2)))
        if many > 1 and rng.random() < 0.5:
            return _case(kind, dtype=dtype, heads=heads, seqs=many, tokens=tokens, **sizes)
        return _case(kind, dtype=dtype, heads=heads, batch=many, length=max(1, tokens // many), **sizes)
    if kind == "pages":
        length = _log_int(rng, 64, 16384)
        return _case(kind, batch=_log_int(rng, 1, 256), page=page, length=length,
                     window=rng.choice([0, 128, 1024, 4096]), sinks=rng.choice([0, 1, 4, 64]),
                     new=rng.choice([1, 1, 4, 16, 160]), spare=rng.choice([30, 95, 100, 130]))
    if kind == "append":
        tokens = _log_int(rng, 1, 8000)
        seqs = _log_int(rng, 1, min(24, tokens))
        return _case(kind, dtype=dtype, heads=heads, seqs=seqs, tokens=tokens, cached=_log_int(rng, 1, 1000), page=page,
                     heads_first=first)
    length = _log_int(rng, 64, 16384)
    batch = _log_int(rng, 1, max(1, min(256, 480000 // length)))
    window = rng.choice([0, 0, 128, 1024, 4096])
    return _case(kind, dtype=dtype, heads=heads, batch=batch, length=length, page=page, draft=rng.choice([1, 1, 1, 2, 4]),
                 window=window, sinks=rng.choice([0, 1, 4, 64]) if window else 0, heads_first=first)


def _lengths(case):
    """Lengths of a packed case's sequences (append: their new tokens), uneven, the same for every seed."""
    n, total = case["seqs"], case["tokens"]
    weights = [1.0 + 7.0 * ((i * 5 + 3) % n) / n for i in range(n)]
    lengths = [max(1, int(total * w / sum(weights))) for w in weights]
    lengths[0] = max(1, lengths[0] + total - sum(lengths))
    return lengths


def _contexts(case):
    """Cached tokens of a decode case's sequences (the query tokens among
    them): the longest first, then uneven ones; of every 50 one is padding."""
    n, longest, draft = case["batch"], case["length"], case["draft"]
    out = [longest]
    for i in range(1, n):
        out.append(0 if i % 50 == 49 else max(draft, longest * (1 + (i * 37) % 97) // 98))
    return out


def _held(case):
    """(tokens cached, new tokens) of a pages case's requests: padding, new prompts, a step's tokens."""
    out = []
    for i in range(case["batch"]):
        cached = case["length"] * (1 + (i * 37) % 97) // 98
        if i % 50 == 49:
            out.append((0, 0))
        elif case["new"] > 16:
            out.append((0, 1 + (i * 53) % case["new"]) if i % 2 else (cached, 1))
        else:
            out.append((cached, 1 + i % case["new"]))
    return out


def _pieces(case):
    """(tokens cached, new tokens) of an append case's sequences; the first of several starts anew."""
    new = _lengths(case)
    return [(0 if i == 0 and len(new) > 1 else 1 + case["cached"] * ((i * 37) % 97) // 97 if i else case["cached"], n)
            for i, n in enumerate(new)]


# ----------------------------------------------------------------------------
# Inputs.
# ----------------------------------------------------------------------------
def _to_fp4(x):
    """x [..., d] -> (bytes [..., d / 2], scales [..., d / 32])."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1)
    code = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)
    m = (x * ((254 - code) << 23).view(torch.float32)[..., None]).abs()
    level = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    level = (level + 8 * (x < 0)).to(torch.uint8).flatten(-2)
    code = torch.where(torch.isfinite(top), code, 255).to(torch.uint8)
    return level[..., 0::2] | (level[..., 1::2] << 4), code


def _from_fp4(data, scale):
    """The float32 values of bytes [..., d / 2] with scales [..., d / 32]."""
    table = torch.tensor([*VALUES, *(-x for x in VALUES)], device=data.device)
    x = table[torch.stack((data & 15, data >> 4), -1).flatten(-2).int()]
    s = (scale.int() << 23).view(torch.float32)
    s = torch.where(scale == 255, math.nan, s)
    return (x.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _caches(case, pages, normal):
    """Two caches of normal values and their scales, [pages, page, hk, ...]; with heads_first
    the heads lie before a page's tokens."""
    page, hk, d = case["page"], case["hk"], case["d"]
    shape = (pages, hk, page) if case["heads_first"] else (pages, page, hk)
    out = []
    for _ in range(2):
        data = torch.empty(*shape, d // 2, dtype=torch.uint8, device="cuda")
        scale = torch.empty(*shape, d // BLOCK, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (page * hk * d))
        for i in range(0, pages, step):
            n = min(step, pages - i)
            data[i:i + n], scale[i:i + n] = _to_fp4(normal(n, *shape[1:], d))
        out += [data.transpose(1, 2), scale.transpose(1, 2)] if case["heads_first"] else [data, scale]
    return dict(k=out[0], v=out[2], k_scale=out[1], v_scale=out[3])


def _table(need, pages, gen):
    """A table with shuffled pages and nothing past each sequence's own, and the pages in their order."""
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, perm[at:]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _rotation(rotary):
    """cos and sin of the rotation's angles, [POSITIONS, rotary / 2]."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, hq, hk, d = DTYPES[case["dtype"]], case["hq"], case["hk"], case["d"]

    def normal(*shape, std=1.0):
        x = torch.empty(shape, dtype=dtype, device="cuda")
        return x.normal_(0.0, std, generator=gen)

    state = dict(case=case, scale=d ** -0.5)
    if case["kind"] in ("rope", "train"):
        packed = "seqs" in case
        batch, length = (1, sum(_lengths(case))) if packed else (case["batch"], case["length"])
        if packed:
            positions = _ints([p for n in _lengths(case) for p in range(n)])
        elif length == 1 or case["kind"] == "rope":  # requests at positions of their own
            start = torch.randint(0, POSITIONS - length, (batch, 1), generator=gen, device="cuda")
            positions = (start + torch.arange(length, device="cuda")).to(torch.int32)
        else:
            positions = torch.arange(length, dtype=torch.int32, device="cuda")
        cos, sin = _rotation(case["rotary"])
        state.update(positions=positions, cos=cos, sin=sin)
        state.update({w: 1.0 + normal(d, std=0.1) for w in ("q_weight", "k_weight")})
        if case["kind"] == "rope":  # columns of one projection's output
            qkv = normal(batch, length, (hq + 2 * hk) * d, std=2.0)
            q, k, _ = qkv.split([hq * d, hk * d, hk * d], -1)
            state.update(q=q.unflatten(-1, (hq, d)), k=k.unflatten(-1, (hk, d)))
            return state
        state.update(q=normal(batch, length, hq, d, std=2.0), k=normal(batch, length, hk, d, std=2.0),
                     grad_q=normal(batch, length, hq, d, std=0.1), grad_k=normal(batch, length, hk, d, std=0.1))
        for name in ("q", "k", "q_weight", "k_weight"):
            state[name].requires_grad_(True)
        return state

    page = case["page"]
    if case["kind"] == "pages":
        held = _held(case)
        rows = [-(-(n + new) // page) for n, new in held]
        wanted = sum(r - -(-n // page) for r, (n, _) in zip(rows, held))
        pool = wanted * case["spare"] // 100
        table, free = _table([-(-n // page) for n, _ in held], sum(-(-n // page) for n, _ in held) + pool, gen)
        wide = torch.full((len(held), max(max(rows), 1) + 3), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        window, kept = case["window"], -(-case["sinks"] // page) * page
        low = [max(kept, n - window) if window else 0 for n, _ in held]  # what the window leaves in this step
        first = [max(kept, x - 4 * page) if window else 0 for x in low]
        free_pages = torch.full((wide.numel() + pool,), -1, dtype=torch.int32, device="cuda")
        free_pages[:pool] = free
        state.update(table=wide, lengths=_ints([n for n, _ in held]), counts=_ints([n for _, n in held]),
                     first=_ints(first), end=_ints(low), free_pages=free_pages, num_free=_ints([pool]),
                     tokens=sum(n for _, n in held))
        return state
    if case["kind"] == "append":
        pieces = _pieces(case)
        need = [-(-(n + new) // page) for n, new in pieces]
        state["table"], _ = _table(need, sum(need) + 3, gen)
        slots = []
        rows = state["table"].tolist()
        for b, (n, new) in enumerate(pieces):
            slots += [rows[b][p // page] * page + p % page for p in range(n, n + new)]
        state.update(slots=_ints(slots, torch.int64), lengths=_ints([n + new for n, new in pieces]), dtype=dtype,
                     tokens=sum(n + new for n, new in pieces), k_new=normal(len(slots), hk, d),
                     v_new=normal(len(slots), hk, d), **_caches(case, sum(need) + 3, normal))
        return state
    contexts = _contexts(case)
    need = [-(-n // page) for n in contexts]
    state["table"], _ = _table(need, sum(need) + 3, gen)
    state.update(lengths=_ints(contexts), q=normal(case["batch"], case["draft"], hq, d),
                 **_caches(case, sum(need) + 3, normal))
    return state


# ----------------------------------------------------------------------------
# One pass.
# ----------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _own(state)
    with torch.no_grad():
        if kind == "rope":
            return tuple(_plain_rope(state[x], state[x + "_weight"], state)[0] for x in ("q", "k"))
        if kind == "train":
            outs = [_plain_rope(state[x], state[x + "_weight"], state, state["grad_" + x]) for x in ("q", "k")]
            return tuple(x for pair in zip(*outs) for x in pair)
        if kind == "pages":
            return _plain_pages(state)
        if kind == "append":
            return _plain_append(state)
        return _plain_decode(state)


def _own(state):
    import pseudobrain_amd as pb
    case = state["case"]
    kind = case["kind"]
    if kind in ("rope", "train"):
        args = tuple(state[x] for x in ("q", "k", "q_weight", "k_weight"))
        if kind == "rope":
            with torch.no_grad():
                return pb.qk_norm_rope(*args, state["cos"], state["sin"], state["positions"], EPS,
                                       interleaved=case["interleaved"])
        q, k = pb.qk_norm_rope(*args, state["cos"], state["sin"], state["positions"], EPS,
                               interleaved=case["interleaved"])
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), args, (state["grad_q"], state["grad_k"]))
    if kind == "pages":
        table, free, page = state["table"], state["free_pages"], case["page"]
        num_free = pb.paged_cache_release(table, state["first"], state["end"], free, state["num_free"], page)
        out = pb.paged_cache_extend(table, state["lengths"], state["counts"], free, num_free, page, state["tokens"])
        return *out, table, free
    cache = (state["k"], state["v"], state["k_scale"], state["v_scale"])
    if kind == "append":
        pb.paged_cache_write_fp4(state["k_new"], state["v_new"], cache, state["slots"])
        return pb.paged_cache_read_fp4(cache, state["table"], state["lengths"], state["tokens"], state["dtype"])
    return pb.paged_decode_attention_fp4(state["q"], cache, state["table"], state["lengths"], state["scale"],
                                         case["window"] or None, case["sinks"])


def _turned(x, cos, sin, interleaved):
    """x [..., d] with its first 2 cos.shape[-1] values rotated in pairs."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rope(x, weight, state, grad=None):
    """The normed and rotated rows; with grad also the gradients of x and the weight."""
    x32, w = x.float(), weight.float()
    at = state["positions"].long()
    cos, sin = state["cos"][at][..., None, :], state["sin"][at][..., None, :]
    if state["positions"].ndim == 1:
        cos, sin = cos[None], sin[None]
    r = torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS)
    interleaved = state["case"]["interleaved"]
    y = _turned(x32 * r * w, cos, sin, interleaved).to(x.dtype)
    if grad is None:
        return (y,)
    g = _turned(grad.float(), cos, -sin, interleaved)
    dw = (g * x32 * r).flatten(0, -2).sum(0)
    g = g * w
    dx = r * (g - x32 * r.square() * (g * x32).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), dw.to(weight.dtype)


def _plain_pages(state):
    table, free, page, tokens = state["table"], state["free_pages"], state["case"]["page"], state["tokens"]
    index = torch.arange(table.shape[1], device="cuda")
    lo, hi = (state[n].long()[:, None] // page for n in ("first", "end"))
    given = (hi - lo).clamp(min=0)
    start = torch.cumsum(given, 0) - given
    to = torch.where((index >= lo) & (index < hi), state["num_free"] + start + index - lo, free.shape[0])
    kept = torch.cat((free, free.new_zeros(1)))
    kept[to.flatten()] = table.flatten()
    free.copy_(kept[:-1])
    num_free = state["num_free"].long() + given.sum()

    lengths, counts = state["lengths"].long(), state["counts"].long()
    held, rows = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    fits = (torch.cumsum(counts, 0) <= tokens) & (rows <= table.shape[1])
    need = torch.where(fits, rows - held, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= num_free))
    counts = torch.where(granted, counts, 0)
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    cu = torch.cat((zero, torch.cumsum(counts, 0)))
    new = granted[:, None] & (index >= held[:, None]) & (index < rows[:, None])
    source = num_free - 1 - ((upto - need - held)[:, None] + index)
    table.copy_(torch.where(new, free[source.clamp(0, free.shape[0] - 1)], table))
    t = torch.arange(tokens, device="cuda")
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=table.shape[0] - 1)
    valid = t < cu[-1]
    position = torch.where(valid, lengths[b] + t - cu[b], 0)
    slot = table[b, position // page].long() * page + position % page
    return (torch.where(valid, slot, -1), torch.where(valid, position, -1).int(), cu.int(), (lengths + counts).int(),
            (num_free - torch.where(granted, need, 0).sum()).int(), table, free)


def _plain_append(state):
    page = state["case"]["page"]
    at = state["slots"]
    for name in ("k", "v"):
        data, scale = _to_fp4(state[name + "_new"])
        state[name][at // page, at % page] = data
        state[name + "_scale"][at // page, at % page] = scale
    cu = torch.cat((state["lengths"].new_zeros(1), torch.cumsum(state["lengths"], 0))).int()
    t = torch.arange(state["tokens"], device="cuda")
    b = torch.searchsorted(cu, t.int(), right=True) - 1
    position = t - cu[b]
    pages = state["table"][b, position // page].long()
    k, v = (_from_fp4(state[n][pages, position % page], state[n + "_scale"][pages, position % page]).to(state["dtype"])
            for n in ("k", "v"))
    return k, v, cu


def _visible(pos, key, window, sinks):
    seen = key <= pos
    if window:
        seen = seen & ((key > pos - window) | (key < sinks))
    return seen


def _plain_decode(state):
    case, scale = state["case"], state["scale"]
    window, sinks, hk, d, page = case["window"], case["sinks"], case["hk"], case["d"], case["page"]
    batch, draft, hq = case["batch"], case["draft"], case["hq"]
    group = hq // hk
    longest = state["table"].shape[1] * page
    if window:  # the keys that any query token sees: the sinks, and the window before the last token
        span = min(longest, window + draft - 1)
        low = (state["lengths"].long() - span).clamp(min=0)
        index = torch.cat([torch.arange(sinks, device="cuda").expand(batch, sinks),
                           low[:, None] + torch.arange(span, device="cuda")], 1)
        once = torch.cat([torch.arange(sinks, device="cuda")[None] < low[:, None],
                          torch.ones(batch, span, dtype=torch.bool, device="cuda")], 1)
    else:
        index = torch.arange(longest, device="cuda").expand(batch, longest)
        once = torch.ones_like(index, dtype=torch.bool)
    out = torch.empty(batch, draft, hq, d, dtype=state["q"].dtype, device="cuda")
    step = max(1, (1 << 28) // (index.shape[1] * hk * d))  # sequences at a time
    for b in range(0, batch, step):
        idx, lens = index[b:b + step], state["lengths"][b:b + step].long()
        n = idx.shape[0]
        held = (idx < lens[:, None]) & once[b:b + step]
        safe = torch.where(held, idx, torch.zeros_like(idx))
        pages, place = state["table"][b:b + step].long().gather(1, safe // page).clamp(min=0), safe % page
        kk, vv = (_from_fp4(state[x][pages, place], state[x + "_scale"][pages, place]).permute(0, 2, 1, 3)
                  for x in ("k", "v"))  # [n, hk, keys, d]
        qq = state["q"][b:b + step].float().view(n, draft, hk, group, d).permute(0, 2, 1, 3, 4)
        pos = (lens[:, None] - draft + torch.arange(draft, device="cuda")).repeat_interleave(group, 1)
        seen = held[:, None, :] & _visible(pos[:, :, None], idx[:, None, :], window, sinks)
        seen = seen[:, None]
        s = torch.matmul(qq.reshape(n, hk, draft * group, d), kk.transpose(2, 3)).mul_(scale)
        s = s.masked_fill_(~seen, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # a row that sees nothing: weights 0
        p = torch.exp(s - top)
        o = torch.matmul(p, vv) / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
        out[b:b + step] = o.view(n, hk, draft, group, d).permute(0, 2, 1, 3, 4).reshape(n, draft, hq, d).to(out.dtype)
    return out


# ----------------------------------------------------------------------------
# What a pass cannot do without.
# ----------------------------------------------------------------------------
def _pairs(queries, keys, window, sinks):
    """Visible (query, key) pairs of the last `queries` positions of `keys` keys."""
    return sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) if window else p + 1
               for p in range(max(0, keys - queries), keys))


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] in ("rope", "train"):
        rows = sum(_lengths(case)) if "seqs" in case else case["batch"] * case["length"]
        values = rows * (hq + hk) * d
        angles = rows if case["kind"] == "rope" else min(rows, case.get("length", rows))
        passes = 2 if case["kind"] == "rope" else 4  # x and y; and the two gradients
        return {"bytes": passes * values * size + angles * case["rotary"] * 4, "flops": (8 if passes == 2 else 24) * values}
    if case["kind"] == "pages":
        page, held = case["page"], _held(case)
        new = sum(-(-(n + m) // page) - -(-n // page) for n, m in held)
        return {"bytes": 12 * sum(m for _, m in held) + 8 * new + 28 * case["batch"], "flops": 0}
    packed = d // 2 + d // BLOCK  # bytes of a head's row in the cache
    if case["kind"] == "append":
        pieces = _pieces(case)
        new, rows = sum(m for _, m in pieces), sum(n + m for n, m in pieces)
        return {"bytes": 2 * hk * (new + rows) * (d * size + packed) + 8 * new, "flops": 0}
    window, sinks = case["window"], case["sinks"]
    pairs = keys = 0
    for n in _contexts(case):
        pairs += _pairs(min(case["draft"], n), n, window, sinks)
        low = max(0, n - window - case["draft"] + 1) if window else 0
        keys += n - low + min(sinks, low)
    rows = case["batch"] * case["draft"] * hq
    return {"bytes": 2 * keys * hk * packed + 2 * rows * d * size, "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------
# From the definitions, in 64 bits.
# ----------------------------------------------------------------------------
def _held_values(data, scale):
    """What bytes and scales stand for, in float64: sign, two bits of exponent, one of mantissa."""
    nibbles = torch.stack((data.long() % 16, data.long() // 16), -1).flatten(-2)
    exponent, mantissa = (nibbles % 8) // 2, (nibbles % 2).double()
    size = torch.where(exponent > 0, (1 + mantissa / 2) * torch.pow(2.0, exponent.double() - 1), mantissa / 2)
    size = torch.where(nibbles >= 8, -size, size)
    return size * torch.pow(2.0, scale.double() - 127).repeat_interleave(BLOCK, -1)


def _nearest(x):
    """x [..., d] in float64 as the cache holds it."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    mantissa, e = torch.frexp(top)  # mantissa in [0.5, 1)
    e = (e - 1 + (mantissa >= 0.875)).clamp(-123, 127)
    s = torch.pow(2.0, torch.where(top > 0, e, -123).double() - 2)
    y, best, at = blocks / s, None, None
    for i in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: they win ties
        far = (y.abs() - VALUES[i]).abs()
        if best is None:
            best, at = far, torch.zeros_like(far)
        else:
            near = far < best
            best, at = torch.where(near, far, best), torch.where(near, VALUES[i], at)
    return (torch.sign(y) * at * s).flatten(-2)


def _exact_rope(x, weight, cos, sin, interleaved):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    half = cos.shape[-1]
    z = y.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        z[..., a] = y[..., a] * cos[..., i] - y[..., b] * sin[..., i]
        z[..., b] = y[..., a] * sin[..., i] + y[..., b] * cos[..., i]
    return z


def _exact_pages(state):
    page, tokens = state["case"]["page"], state["tokens"]
    table, free = state["table"].tolist(), state["free_pages"].tolist()
    num_free = int(state["num_free"])
    for b, (lo, hi) in enumerate(zip(state["first"].tolist(), state["end"].tolist())):
        for i in range(len(table[b])):
            if lo <= i * page + page - 1 < hi:
                free[num_free] = table[b][i]
                num_free += 1
    slots, positions, cu, lengths = [], [], [0], []
    asked, wanted, pool = 0, 0, num_free
    for b, (n, new) in enumerate(zip(state["lengths"].tolist(), state["counts"].tolist())):
        asked += new
        held, rows = -(-n // page), -(-(n + new) // page)
        ok = asked <= tokens and rows <= len(table[b])
        wanted += rows - held if ok else 0
        ok = ok and (rows == held or wanted <= pool)
        if ok:
            for i in range(held, rows):
                num_free -= 1
                table[b][i] = free[num_free]
            for p in range(n, n + new):
                slots.append(table[b][p // page] * page + p % page)
                positions.append(p)
        cu.append(len(slots))
        lengths.append(n + new if ok else n)
    pad = [-1] * (tokens - len(slots))
    return (_ints(slots + pad, torch.int64), _ints(positions + pad), _ints(cu), _ints(lengths), _ints([num_free]),
            _ints(table), _ints(free))


def exact(case, seed):
    state = prepare(case, seed)
    kind, scale = case["kind"], state["scale"]
    if kind in ("rope", "train"):
        at = state["positions"].long()
        cos, sin = (state[n].double()[at].unsqueeze(-2) for n in ("cos", "sin"))
        names = ("q", "k", "q_weight", "k_weight")
        inputs = [state[n].detach().double().requires_grad_(kind == "train") for n in names]
        outs = [_exact_rope(inputs[i], inputs[2 + i], cos, sin, case["interleaved"]) for i in range(2)]
        if kind == "rope":
            return tuple(outs)
        grads = torch.autograd.grad(outs, inputs, [state["grad_q"].double(), state["grad_k"].double()])
        return *(x.detach() for x in outs), *grads
    if kind == "pages":
        return _exact_pages(state)
    page, hk, d = case["page"], case["hk"], case["d"]
    table = state["table"].cpu()
    if kind == "append":
        outs, cu = ([], []), [0]
        new = 0
        for b, (cached, n) in enumerate(_pieces(case)):
            pages = table[b, :-(-(cached + n) // page)].long().cuda()
            for out, name in zip(outs, ("k", "v")):
                rows = _held_values(state[name][pages], state[name + "_scale"][pages]).flatten(0, 1)[:cached + n]
                rows[cached:] = _nearest(state[name + "_new"][new:new + n].double())
                out.append(rows)
            new += n
            cu.append(cu[-1] + cached + n)
        return torch.cat(outs[0]), torch.cat(outs[1]), _ints(cu)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_contexts(case)):
        if n == 0:
            continue
        pages = table[b, :-(-n // page)].long().cuda()
        k, v = (_held_values(state[x][pages], state[x + "_scale"][pages]).flatten(0, 1)[:n] for x in ("k", "v"))
        distance = (torch.arange(n - case["draft"], n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None])
        hidden = distance < 0
        if case["window"]:
            hidden = hidden | ((distance >= case["window"]) & (torch.arange(n, device="cuda") >= case["sinks"])[None])
        for h in range(hk):
            group = case["hq"] // hk
            q = state["q"][b, :, h * group:(h + 1) * group].double()  # [draft, group, d]
            logits = (scale * (q.reshape(-1, d) @ k[:, h].t())).view(case["draft"], group, n)
            p = torch.softmax(logits.masked_fill(hidden[:, None], -math.inf), -1)
            out[b, :, h * group:(h + 1) * group] = (p.view(-1, n) @ v[:, h]).view(case["draft"], group, d)
    return out
