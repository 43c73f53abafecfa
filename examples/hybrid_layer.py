"""A hybrid layer's mixer on the device: a Gated DeltaNet recurrence and windowed
attention over the same tokens, their outputs summed
(WindowedHybridLayer.mix, pseudobrain/transplant.py:989-997), in the three
ways a model uses it:

  train    forward and backward of a batch (gated_delta_rule, window_attention)
  prefill  a prompt into the recurrent state and the paged key-value cache
           (chunk_fwd_slots, window_attention, paged_cache_write)
  decode   one token a step against both (recurrent_step_, paged_cache_write,
           paged_decode_attention), pages left of the window given back

    python examples/hybrid_layer.py

Weights and tokens are random; the last line compares the decoded tokens'
outputs with one pass over the whole sequence.
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pseudobrain_amd import (chunk_fwd_slots, gated_delta_rule, paged_cache_write, paged_decode_attention,  # noqa: E402
                             window_attention)

HIDDEN, HQ, HK, D, V_HEADS = 512, 8, 2, 64, 4  # query, key heads and width of both halves; the recurrence's value heads
WINDOW, SINKS, PAGE = 64, 4, 16
SCALE = D ** -0.5


class Mixer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.widths = [HQ * D, HK * D, HK * D, HK * D, HK * D, V_HEADS * D, V_HEADS, V_HEADS]
        self.proj = torch.nn.Linear(HIDDEN, sum(self.widths), bias=False)

    def split(self, x):
        """x [B,T,HIDDEN] -> attention's q, k, v and the recurrence's q, k, v, g, beta."""
        parts = self.proj(x).split(self.widths, -1)
        q, k, v, rq, rk, rv = (p.unflatten(-1, (-1, D)) for p in parts[:6])
        g, beta = -F.softplus(parts[6].float()), torch.sigmoid(parts[7].float())
        return (q, k, v), (F.normalize(rq, dim=-1), F.normalize(rk, dim=-1), rv, g, beta)

    def forward(self, x):
        (q, k, v), rec = self.split(x)
        state = torch.zeros(x.shape[0], V_HEADS, D, D, device=x.device)
        o, _ = gated_delta_rule(*rec, SCALE, state, "hip")
        a = window_attention(q, k, v, SCALE, WINDOW, SINKS)
        return torch.cat([a.flatten(2).float(), o.flatten(2)], -1)  # the layer's output projection sums the halves


class Cache:
    """One sequence's memory: a state slot, and pages taken from a pool as it grows."""

    def __init__(self, tokens: int, device):
        pages = -(-tokens // PAGE)
        self.k, self.v = (torch.zeros(pages + 2, PAGE, HK, D, dtype=torch.bfloat16, device=device) for _ in range(2))
        self.state = torch.zeros(1, V_HEADS, D, D, device=device)
        self.slot = torch.zeros(1, dtype=torch.int32, device=device)
        self.table = torch.full((1, pages), -1, dtype=torch.int32, device=device)
        self.free = torch.randperm(pages + 2).tolist()
        self.pages, self.length = [], 0  # the sequence's pages in order, None where given back

    def extend(self, n: int) -> torch.Tensor:
        """Slots of n more tokens. Pages that neither hold sinks nor any key the newest
        token sees are given back."""
        while len(self.pages) * PAGE < self.length + n:
            self.table[0, len(self.pages)] = self.free[-1]
            self.pages.append(self.free.pop())
        at = [self.pages[j // PAGE] * PAGE + j % PAGE for j in range(self.length, self.length + n)]
        self.length += n
        for i in range(-(-SINKS // PAGE), max(0, self.length - WINDOW) // PAGE):
            if self.pages[i] is not None:
                self.free.append(self.pages[i])
                self.pages[i], self.table[0, i] = None, -1
        return torch.tensor(at, device=self.k.device)


@torch.no_grad()
def prefill(mixer, x, cache):
    (q, k, v), rec = mixer.split(x)
    o = chunk_fwd_slots(*rec, SCALE, cache.state, cache.slot, out_dtype=torch.float32)
    a = window_attention(q, k, v, SCALE, WINDOW, SINKS)
    paged_cache_write(k[0], v[0], cache.k, cache.v, cache.extend(x.shape[1]))
    return torch.cat([a.flatten(2).float(), o.flatten(2)], -1)


@torch.no_grad()
def decode(mixer, x, cache):
    (q, k, v), rec = mixer.split(x)
    o = torch.ops.pbgdn.recurrent_step_(*rec, cache.state, cache.slot, SCALE)
    paged_cache_write(k[0], v[0], cache.k, cache.v, cache.extend(1))
    lengths = torch.tensor([cache.length], dtype=torch.int32, device=x.device)
    a = paged_decode_attention(q, cache.k, cache.v, cache.table, lengths, SCALE, WINDOW, SINKS)
    return torch.cat([a.flatten(2).float(), o.float().flatten(2)], -1)


def run(prompt: int = 300, new: int = 50, device="cuda"):
    """Trains one step, then serves a prompt and `new` tokens. Returns the loss, the
    weights' gradient, and the served outputs beside those of one pass."""
    torch.manual_seed(0)
    mixer = Mixer().to(device, torch.bfloat16)
    x = torch.randn(1, prompt + new, HIDDEN, device=device).to(torch.bfloat16)
    loss = mixer(x).square().mean()
    loss.backward()
    with torch.no_grad():
        whole = mixer(x)
    cache = Cache(prompt + new, device)
    served = [prefill(mixer, x[:, :prompt], cache)]
    served += [decode(mixer, x[:, t:t + 1], cache) for t in range(prompt, prompt + new)]
    return loss.item(), mixer.proj.weight.grad, torch.cat(served, 1), whole, cache


if __name__ == "__main__":
    loss, grad, served, whole, cache = run()
    print(f"loss {loss:.4f}, gradient norm {grad.float().norm().item():.3e}")
    print(f"{cache.length} tokens served, {len(cache.pages) - cache.pages.count(None)} of {len(cache.pages)} pages held")
    print(f"largest difference from one pass over the sequence: {(served - whole).abs().max().item():.2e} "
          f"of outputs up to {whole.abs().max().item():.2f}")
