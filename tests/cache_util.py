"""Helpers for the tests of the rotary and cache operators: caches of every layout, and the operators in 64 bits on the CPU."""
from __future__ import annotations

import math
import random

import torch

BF16_HALF_STEP = torch.finfo(torch.bfloat16).eps / 2     # a rounding to bf16 is off by at most this share of the value


def randn(gen, *shape):
    return torch.randn(*shape, generator=gen).to(torch.bfloat16)


class Cache:
    """A cache on the GPU with random contents, and where each sequence's slots are.

    ``page`` 0: one piece a sequence.  ``layout``: "plain" [pages, page, heads, 128]; "pairs": k and v of a page side by
    side; "heads": heads before slots; "layers": one layer of three.
    """

    def __init__(self, seed, seqs, slots, kvh, page=0, layout="plain", device="cuda"):
        gen = torch.Generator().manual_seed(seed + 77777)     # a stream of its own: no key equals a query
        self.kvh, self.page, self.seqs = kvh, page, seqs
        width = 1 if page == 0 else -(-slots // page)
        size = slots if page == 0 else page
        pages = seqs if page == 0 else seqs * width + 2
        self.slots = width * size
        if layout == "pairs":
            pool = randn(gen, pages, 2, size, kvh, 128).to(device)
            self.k, self.v = pool[:, 0], pool[:, 1]
        elif layout == "heads":
            self.k, self.v = (randn(gen, pages, kvh, size, 128).to(device).transpose(1, 2) for _ in range(2))
        elif layout == "layers":
            pool = randn(gen, 2, pages, size, 3, kvh, 128).to(device)
            self.k, self.v = pool[0, :, :, 1], pool[1, :, :, 1]
        else:
            self.k, self.v = (randn(gen, pages, size, kvh, 128).to(device) for _ in range(2))
        if page == 0:
            self.table = None
            self.place = [[(b, s) for s in range(slots)] for b in range(seqs)]
        else:
            order = list(range(pages))
            random.Random(seed).shuffle(order)
            table = [order[b * width:(b + 1) * width] for b in range(seqs)]
            self.table = torch.tensor(table, dtype=torch.int32).to(device)
            self.place = [[(table[b][s // page], s % page) for s in range(width * page)] for b in range(seqs)]

    def index(self, b, first=0, last=None):
        """(pages, rows) of slots [first, last) of sequence b, for indexing k or v."""
        at = self.place[b][first:last]
        return torch.tensor([p for p, _ in at], dtype=torch.long), torch.tensor([r for _, r in at], dtype=torch.long)

    def rows(self, which, b, n):
        """The first n slots of sequence b, [n, heads, 128] in 64 bits on the CPU."""
        cache = getattr(self, which)
        pages, rows = self.index(b, 0, n)
        return cache[pages.to(cache.device), rows.to(cache.device)].double().cpu()


def turn(x, positions, freq, axis, adjacent, sign=1):
    """x [tokens, heads, 128] turned in 64 bits: pairs as complex numbers."""
    pairs = len(freq)
    x = x.double()
    first = torch.arange(pairs) * 2 if adjacent else torch.arange(pairs)
    second = first + 1 if adjacent else first + pairs
    angle = torch.stack([positions[a].double() * f for f, a in zip(freq, axis)], 1)[:, None]
    out = x.clone()
    a, b = x[:, :, first], x[:, :, second]
    out[:, :, first] = a * angle.cos() - sign * b * angle.sin()
    out[:, :, second] = b * angle.cos() + sign * a * angle.sin()
    return out


def assert_turned(ours, x, ref, pairs):
    """One rounding to bf16 (half a step of the result), and sin, cos, two products and a sum in 32 bits: each is off by at most
    2^-23 or so of a term, which is at most the pair's length; 2^-20 of the largest value covers them."""
    ours, ref = ours.double().cpu(), ref.cpu()
    slack = ref.abs() * BF16_HALF_STEP * (1 + 2**-10) + 2**-20 * x.double().abs().max().item()
    bad = (ours - ref).abs() > slack
    assert not bad.any(), f"{int(bad.sum())} values off, the worst by {(ours - ref).abs().max().item():.3e}"
    assert torch.equal(ours[..., 2 * pairs:], x.double().cpu()[..., 2 * pairs:]), "dimensions behind the pairs changed"


def ancestors(rng, count):
    """Masks of a random tree: [count, count], a token sees itself and its ancestors."""
    seen = torch.zeros(count, count, dtype=torch.bool)
    for i in range(count):
        parent = rng.randint(max(-1, i // 2 - 2), i - 1)
        if parent >= 0:
            seen[i] = seen[parent]
        seen[i, i] = True
    return seen


def tree_attention(q, k, v, seen):
    """One sequence in 64 bits: q [n, QH, 128], k, v [slots, KVH, 128], seen [n, slots] -> out [n, QH, 128], lse [QH, n], and
    the root of the sum of the squares of out's terms.  What a row does not see has no part in it, whatever it is."""
    group = q.size(1) // k.size(1)
    q, k, v = q.double(), k.double(), v.double()
    out, spread, lse = torch.zeros_like(q), torch.zeros_like(q), torch.full((q.size(1), q.size(0)), -math.inf, dtype=torch.float64)
    for i in range(q.size(0)):
        if not seen[i].any():
            continue
        ki, vi = k[seen[i]].repeat_interleave(group, 1), v[seen[i]].repeat_interleave(group, 1)
        s = torch.einsum("hd,shd->hs", q[i], ki) / math.sqrt(128)
        lse[:, i] = s.logsumexp(1)
        p = s.softmax(1)
        out[i] = torch.einsum("hs,shd->hd", p, vi)
        spread[i] = torch.einsum("hs,shd->hd", p * p, vi * vi).sqrt()
    return out, lse, spread
