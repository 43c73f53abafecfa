"""The workloads by which the attention operators' speed is judged: the windowed
attention half of a hybrid layer, whose other half is the Gated DeltaNet
recurrence, in training, prefill and decode.

Four kinds of call:

  prefill  window_attention without gradients: one prompt, packed prompts
  train    window_attention and its backward through autograd
  decode   paged_decode_attention: the newest token (or the sampled token and
           the drafted ones) of each running request against a paged cache
  write    paged_cache_write: new keys and values into the cache's pages

A query at position p sees key j when j <= p and (j > p - window or j < sinks);
window 0 means no window. hq query heads share hk key heads in groups.

A case is a dict of plain values:
  kind, dtype, hq, hk, d, window, sinks
  batch, length   (prefill, train: unpacked)
  seqs, tokens    (prefill, train: that many sequences of uneven lengths in all `tokens`)
  batch, length, page, draft   (decode: the longest sequence, tokens a page, query tokens a sequence)
  tokens, page    (write)
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
WIDE = dict(hq=32, hk=8, d=128)    # grouped heads of the usual width
K256 = dict(hq=16, hk=2, d=256)    # the widest heads, eight queries to a key head
SMALL = dict(hq=4, hk=4, d=64)     # the small float32 model: a key head for each query head
ROWS = 1024                        # query rows the plain form handles at a time


def _case(kind, dtype="bfloat16", heads=None, window=0, sinks=0, **sizes):
    return dict(kind=kind, dtype=dtype, **(WIDE if heads is None else heads), window=window, sinks=sinks, **sizes)


def listed():
    return [
        # a single chat prompt: one sequence shorter than its window
        dict(_case("prefill", window=1024, sinks=4, batch=1, length=777), name="prefill_chat_777"),
        # one long document through the window
        dict(_case("prefill", window=4096, sinks=4, batch=1, length=32768), name="prefill_32768_w4096"),
        # a serving engine's prefill batch of uneven prompts, widest heads
        dict(_case("prefill", heads=K256, window=1024, sinks=64, seqs=24, tokens=19001), name="prefill_k256_24seq"),
        # the small model in float32, every earlier token visible
        dict(_case("prefill", dtype="float32", heads=SMALL, batch=1, length=2048), name="prefill_small_fp32"),
        # a training batch
        dict(_case("train", window=1024, sinks=4, batch=4, length=2048), name="train_4x2048_w1024"),
        # long-context training, every earlier token visible, float16
        dict(_case("train", dtype="float16", batch=1, length=8192), name="train_1x8192_fp16"),
        # packed training documents of uneven lengths, widest heads
        dict(_case("train", heads=K256, window=512, sinks=4, seqs=7, tokens=6011), name="train_k256_7seq"),
        # one user at the keyboard: latency only
        dict(_case("decode", batch=1, length=4097, page=16, draft=1), name="decode_b1_4097"),
        # a steady serving batch of uneven contexts without a window
        dict(_case("decode", batch=64, length=16384, page=16, draft=1), name="decode_b64_16384"),
        # a full serving batch of an odd size: window and sinks, four tokens to verify, large pages of no round size
        dict(_case("decode", heads=K256, window=4096, sinks=64, batch=233, length=8192, page=528, draft=4),
             name="decode_k256_b233_w4096"),
        # the new tokens of a decode step
        dict(_case("write", tokens=64, page=16), name="write_64"),
        # the tokens of a prefill batch
        dict(_case("write", heads=K256, tokens=19001, page=528), name="write_k256_19001"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed kinds' ranges, none dearer than the dearest listed."""
    kind = rng.choice(["prefill", "prefill", "train", "train", "decode", "decode", "write"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    heads = rng.choice([WIDE, K256, dict(hq=24, hk=8, d=64), dict(hq=16, hk=16, d=128), dict(hq=14, hk=2, d=128)])
    if dtype == "float32":
        heads = rng.choice([SMALL, dict(hq=8, hk=2, d=128)])
    page = rng.choice([16, 32, 64, 100, 528])
    sinks = rng.choice([0, 1, 4, 64])
    if kind == "write":
        return _case(kind, dtype=dtype, heads=heads, tokens=_log_int(rng, 1, 19001), page=page)
    if kind == "decode":
        length = _log_int(rng, 64, 16384)
        batch = _log_int(rng, 1, max(1, min(256, 480000 // length)))
        window = rng.choice([0, 0, 128, 1024, 4096])
        return _case(kind, dtype=dtype, heads=heads, window=window, sinks=sinks if window else 0, batch=batch,
                     length=length, page=page, draft=rng.choice([1, 1, 1, 2, 4]))
    top = 8192 if dtype == "float32" else 15000 if kind == "prefill" else 8192
    tokens = _log_int(rng, 17, top)
    window = rng.choice([0, 128, 512, 1000, 1024, 4096])
    sizes = dict(window=window, sinks=sinks if window else 0)
    many = _log_int(rng, 1, min(24, max(1, tokens // 16)))
    if many > 1 and rng.random() < 0.5:
        return _case(kind, dtype=dtype, heads=heads, seqs=many, tokens=tokens, **sizes)
    return _case(kind, dtype=dtype, heads=heads, batch=many, length=max(5, tokens // many), **sizes)


def _lengths(case):
    """Lengths of a packed case's sequences, uneven, the same for every seed."""
    n, total = case["seqs"], case["tokens"]
    weights = [1.0 + 7.0 * ((i * 5 + 3) % n) / n for i in range(n)]
    lengths = [max(1, int(total * w / sum(weights))) for w in weights]
    lengths[0] += total - sum(lengths)
    return lengths


def _contexts(case):
    """Cached tokens of a decode case's sequences (the query tokens among
    them): the longest first, then uneven ones; of every 50 one is padding."""
    n, longest, draft = case["batch"], case["length"], case["draft"]
    out = [longest]
    for i in range(1, n):
        out.append(0 if i % 50 == 49 else max(draft, longest * (1 + (i * 37) % 97) // 98))
    return out


def _spans(case):
    """(first token, length) of each sequence in a prefill or train case's flattened tokens."""
    lengths = _lengths(case) if "seqs" in case else [case["length"]] * case["batch"]
    start, out = 0, []
    for n in lengths:
        out.append((start, n))
        start += n
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, hq, hk, d = DTYPES[case["dtype"]], case["hq"], case["hk"], case["d"]

    def normal(*shape, std=1.0):
        x = torch.empty(shape, dtype=dtype, device="cuda")
        return x.normal_(0.0, std, generator=gen)

    state = dict(case=case, scale=d ** -0.5)
    if case["kind"] in ("prefill", "train"):
        packed = "seqs" in case
        batch, length = (1, case["tokens"]) if packed else (case["batch"], case["length"])
        state.update(q=normal(batch, length, hq, d), k=normal(batch, length, hk, d), v=normal(batch, length, hk, d))
        if packed:
            cu = [s for s, _ in _spans(case)] + [length]
            state["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        else:
            state["cu"] = None
        if case["kind"] == "train":
            state["grad_o"] = normal(batch, length, hq, d, std=0.1)
            for name in ("q", "k", "v"):
                state[name].requires_grad_(True)
        return state

    page = case["page"]
    if case["kind"] == "decode":
        contexts = _contexts(case)
        need = [-(-n // page) for n in contexts]
        pages = sum(need) + 3
        perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n]
            at += n
        state.update(table=table, lengths=torch.tensor(contexts, dtype=torch.int32, device="cuda"),
                     q=normal(case["batch"], case["draft"], hq, d))
    else:
        tokens = case["tokens"]
        pages = -(-tokens // page) + 5
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens]
        slots[tokens // 2::97] = -1  # padding tokens, which are not written
        state.update(slots=slots, k=normal(tokens, hk, d), v=normal(tokens, hk, d))
    state.update(k_cache=normal(pages, page, hk, d), v_cache=normal(pages, page, hk, d))
    return state


# ----------------------------------------------------------------------------
# One pass.
# ----------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind, window, sinks = case["kind"], case["window"], case["sinks"]
    if own:
        from pseudobrain_amd.attention import paged_cache_write, paged_decode_attention, window_attention
        if kind == "prefill":
            with torch.no_grad():
                return window_attention(state["q"], state["k"], state["v"], state["scale"], window or None, sinks,
                                        state["cu"])
        if kind == "train":
            q, k, v = state["q"], state["k"], state["v"]
            o = window_attention(q, k, v, state["scale"], window or None, sinks, state["cu"])
            return (o.detach(), *torch.autograd.grad(o, (q, k, v), state["grad_o"]))
        if kind == "decode":
            return paged_decode_attention(state["q"], state["k_cache"], state["v_cache"], state["table"],
                                          state["lengths"], state["scale"], window or None, sinks)
        paged_cache_write(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"])
        return state["k_cache"], state["v_cache"]
    with torch.no_grad():
        if kind == "prefill":
            return _plain_attention(state, None)[0]
        if kind == "train":
            return _plain_attention(state, state["grad_o"])
        if kind == "decode":
            return _plain_decode(state)
        return _plain_write(state)


def _visible(pos, key, window, sinks):
    seen = key <= pos
    if window:
        seen = seen & ((key > pos - window) | (key < sinks))
    return seen


def _plain_attention(state, grad_o):
    """Blocks of query rows against the keys that any of them sees. With grad_o
    also the gradients of q, k and v."""
    case, scale = state["case"], state["scale"]
    window, sinks, hk = case["window"], case["sinks"], case["hk"]
    group, d = case["hq"] // hk, case["d"]
    shape, kv_shape = state["q"].shape, state["k"].shape
    q, k, v = (state[n].float().view(-1, h, d) for n, h in (("q", hk * group), ("k", hk), ("v", hk)))
    o = torch.zeros_like(q)
    if grad_o is not None:
        go = grad_o.float().view(-1, hk * group, d)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)

    def rows(x, at, n):  # [tokens, heads, d] -> [hk, n * group, d], the heads of a group together
        return x[at:at + n].view(n, hk, group, d).permute(1, 0, 2, 3).reshape(hk, n * group, d)

    def tokens(x, n):
        return x.view(hk, n, group, d).permute(1, 0, 2, 3).reshape(n, hk * group, d)

    for start, length in _spans(case):
        for first in range(0, length, ROWS):
            n = min(ROWS, length - first)
            low = max(0, first - window + 1) if window else 0
            keys = torch.arange(low, first + n, device=q.device)
            if window:
                keys = torch.cat([torch.arange(min(sinks, low), device=q.device), keys])
            at = keys + start
            kk, vv = k[at].transpose(0, 1), v[at].transpose(0, 1)  # [hk, keys, d]
            pos = torch.arange(first, first + n, device=q.device).repeat_interleave(group)
            seen = _visible(pos[:, None], keys[None, :], window, sinks)
            qq = rows(q, start + first, n)
            s = torch.matmul(qq, kk.transpose(1, 2)).mul_(scale).masked_fill_(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            out = torch.matmul(p, vv)
            o[start + first:start + first + n] = tokens(out, n)
            if grad_o is None:
                continue
            gg = rows(go, start + first, n)
            dv.index_add_(0, at, torch.matmul(p.transpose(1, 2), gg).transpose(0, 1).contiguous())
            ds = p * (torch.matmul(gg, vv.transpose(1, 2)) - (gg * out).sum(-1, keepdim=True)) * scale
            dk.index_add_(0, at, torch.matmul(ds.transpose(1, 2), qq).transpose(0, 1).contiguous())
            dq[start + first:start + first + n] = tokens(torch.matmul(ds, kk), n)
    dtype = state["q"].dtype
    o = o.view(shape).to(dtype)
    if grad_o is None:
        return (o,)
    return o, dq.view(shape).to(dtype), dk.view(kv_shape).to(dtype), dv.view(kv_shape).to(dtype)


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
        slot = state["table"][b:b + step].long().gather(1, safe // page).clamp(min=0) * page + safe % page
        kk = state["k_cache"].view(-1, hk, d)[slot].float().permute(0, 2, 1, 3)  # [n, hk, keys, d]
        vv = state["v_cache"].view(-1, hk, d)[slot].float().permute(0, 2, 1, 3)
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


def _plain_write(state):
    kept = state["slots"] >= 0
    at = state["slots"][kept]
    k_cache, v_cache = state["k_cache"], state["v_cache"]
    k_cache.view(-1, *k_cache.shape[2:])[at] = state["k"][kept]
    v_cache.view(-1, *v_cache.shape[2:])[at] = state["v"][kept]
    return k_cache, v_cache


# ----------------------------------------------------------------------------
# What a pass cannot do without.
# ----------------------------------------------------------------------------
def _pairs(queries, keys, window, sinks):
    """Visible (query, key) pairs of the last `queries` positions of `keys` keys."""
    total = 0
    first = keys - queries
    full = min(max(window, 0), keys) if window else keys
    for p in range(max(0, first), min(keys, full)):  # positions that see every earlier key
        total += p + 1
    if window:
        start = max(first, full, 0)
        # from position `window` on: the window, and the sinks to its left
        left = [min(sinks, p - window + 1) for p in range(start, min(keys, window + sinks))]
        rest = max(0, keys - max(start, window + sinks))
        total += (keys - start) * window + sum(left) + rest * sinks if keys > start else 0
    return total


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    hq, hk, d = case["hq"], case["hk"], case["d"]
    window, sinks = case["window"], case["sinks"]
    if case["kind"] == "write":
        kept = case["tokens"] - len(range(case["tokens"] // 2, case["tokens"], 97))
        return {"bytes": 4 * kept * hk * d * size + 8 * case["tokens"], "flops": 0}
    if case["kind"] == "decode":
        pairs = keys = 0
        for n in _contexts(case):
            pairs += _pairs(min(case["draft"], n), n, window, sinks)
            if window:
                low = max(0, n - window - case["draft"] + 1)
                keys += n - low + min(sinks, low)
            else:
                keys += n
        rows = case["batch"] * case["draft"] * hq
        return {"bytes": (2 * keys * hk + 2 * rows) * d * size, "flops": 4 * d * hq * pairs}
    spans = _spans(case)
    tokens = sum(n for _, n in spans)
    pairs = hq * sum(_pairs(n, n, window, sinks) for _, n in spans)
    if case["kind"] == "prefill":
        return {"bytes": tokens * (2 * hq + 2 * hk) * d * size, "flops": 4 * d * pairs}
    return {"bytes": tokens * (4 * hq + 4 * hk) * d * size, "flops": 14 * d * pairs}


# ----------------------------------------------------------------------------
# From the definition, in 64 bits.
# ----------------------------------------------------------------------------
def _exact_head(q, k, v, first, window, sinks, scale):
    """Attention of one head in float64: q [n, d] at positions first.., k and v [m, d]."""
    pos = first + torch.arange(q.shape[0], device=q.device)
    dist = pos[:, None] - torch.arange(k.shape[0], device=q.device)[None, :]
    hidden = dist < 0
    if window:
        hidden = hidden | ((dist >= window) & (torch.arange(k.shape[0], device=q.device) >= sinks)[None, :])
    logits = (scale * (q @ k.t())).masked_fill(hidden, -math.inf)
    return torch.softmax(logits, -1) @ v


def exact(case, seed):
    state = prepare(case, seed)
    window, sinks, scale = case["window"], case["sinks"], state["scale"]
    group = case["hq"] // case["hk"]
    if case["kind"] == "write":
        caches = []
        for name in ("k", "v"):
            cache = state[name + "_cache"].double()
            flat = cache.view(-1, case["hk"], case["d"])
            index = state["slots"].tolist()
            src = torch.tensor([i for i, s in enumerate(index) if s >= 0], device="cuda")
            dst = torch.tensor([s for s in index if s >= 0], device="cuda")
            flat.index_copy_(0, dst, state[name].double().index_select(0, src))
            caches.append(cache)
        return tuple(caches)
    if case["kind"] == "decode":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        table = state["table"].cpu()
        for b, n in enumerate(_contexts(case)):
            if n == 0:
                continue
            pages = table[b, :-(-n // case["page"])].long().cuda()
            k = state["k_cache"][pages].double().flatten(0, 1)[:n]
            v = state["v_cache"][pages].double().flatten(0, 1)[:n]
            for h in range(case["hq"]):
                out[b, :, h] = _exact_head(state["q"][b, :, h].double(), k[:, h // group], v[:, h // group],
                                           n - case["draft"], window, sinks, scale)
        return out
    d, train = case["d"], case["kind"] == "train"
    q, k, v = (state[n].detach().double().flatten(0, 1) for n in ("q", "k", "v"))
    outs = [torch.zeros_like(x) for x in ((q, q, k, v) if train else (q,))]
    block = 2048
    for start, length in _spans(case):
        for h in range(case["hq"]):
            kh = k[start:start + length, h // group].requires_grad_(train)
            vh = v[start:start + length, h // group].requires_grad_(train)
            for first in range(0, length, block):
                rows = slice(start + first, start + min(length, first + block))
                last = min(length, first + block)
                qh = q[rows, h].requires_grad_(train)
                o = _exact_head(qh, kh[:last], vh[:last], first, window, sinks, scale)
                outs[0][rows, h] = o.detach()
                if train:
                    grad_o = state["grad_o"].flatten(0, 1)[rows, h].double()
                    dq, dk, dv = torch.autograd.grad(o, (qh, kh, vh), grad_o)
                    outs[1][rows, h] = dq
                    outs[2][start:start + length, h // group] += dk
                    outs[3][start:start + length, h // group] += dv
    shapes = [state[n].shape for n in ("q", "q", "k", "v")]
    outs = [x.view(s) for x, s in zip(outs, shapes)]
    return tuple(outs) if train else outs[0]
