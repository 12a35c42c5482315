"""Helpers for the tests of caches in 8 bits: caches of every layout, rounding to e4m3 and the writing of blocks in 64 bits on the CPU."""
from __future__ import annotations

import math
import random

import torch

E4M3 = torch.float8_e4m3fn
E4M3_HALF_STEP = torch.finfo(E4M3).eps / 2       # a rounding to e4m3 is off by at most this share of the value,
E4M3_SMALLEST = 2.0**-9                          # or by half of this below 2^-6


def to_e4m3(x):
    """64-bit values rounded to e4m3: to a multiple of an eighth of their power of two, of 2^-9 at least, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-40))).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def scale_for(most):
    """The smallest power of two, from 2^-64 to 2^64, of which ``most`` is at most 448 times."""
    if most == 0:
        return 2.0**-64
    e = math.frexp(most / 448)[1]                # most / 448 = m 2^e, m in [0.5, 1)
    return 2.0 ** max(-64, min(64, e - 1 if math.ldexp(0.5, e) == most / 448 else e))


class Cache8:
    """A cache on the GPU with random contents and scales, and where each sequence's slots are.

    ``page`` 0: one piece a sequence.  ``layout``: "plain" [pages, page, heads, 128]; "pairs": k and v of a page side by
    side, their scales likewise; "heads": heads before slots, in the scales too; "layers": one layer of three.
    ``spread``: how many powers of two the scales of blocks differ by; ``powers``: scales are powers of two.
    """

    def __init__(self, seed, seqs, slots, kvh, page=0, block=16, layout="plain", spread=3, powers=True, device="cuda"):
        gen = torch.Generator().manual_seed(seed + 99999)
        self.kvh, self.page, self.block, self.seqs = kvh, page, block, seqs
        width = 1 if page == 0 else -(-slots // page)
        size = slots if page == 0 else page
        pages = seqs if page == 0 else seqs * width + 2
        blocks = -(-size // block)
        self.slots = width * size

        def contents(*shape):
            return (torch.randn(*shape, generator=gen) * 100).clamp(-448, 448).to(E4M3).to(device)

        def scales(*shape):
            e = torch.rand(*shape, generator=gen) * spread - 7 - spread / 2
            return torch.exp2(e.round() if powers else e).float().to(device)

        if layout == "pairs":
            pool, both = contents(pages, 2, size, kvh, 128), scales(pages, 2, blocks, kvh)
            self.k, self.v, self.k_scales, self.v_scales = pool[:, 0], pool[:, 1], both[:, 0], both[:, 1]
        elif layout == "heads":
            self.k, self.v = (contents(pages, kvh, size, 128).transpose(1, 2) for _ in range(2))
            self.k_scales, self.v_scales = (scales(pages, kvh, blocks).transpose(1, 2) for _ in range(2))
        elif layout == "layers":
            pool, both = contents(2, pages, size, 3, kvh, 128), scales(2, pages, 3, blocks, kvh)
            self.k, self.v, self.k_scales, self.v_scales = pool[0, :, :, 1], pool[1, :, :, 1], both[0, :, 1], both[1, :, 1]
        else:
            self.k, self.v = (contents(pages, size, kvh, 128) for _ in range(2))
            self.k_scales, self.v_scales = (scales(pages, blocks, kvh) for _ in range(2))
        if page == 0:
            self.table = None
            self.place = [[(b, s) for s in range(slots)] for b in range(seqs)]
        else:
            order = list(range(pages))
            random.Random(seed).shuffle(order)
            table = [order[b * width:(b + 1) * width] for b in range(seqs)]
            self.table = torch.tensor(table, dtype=torch.int32).to(device)
            self.place = [[(table[b][s // page], s % page) for s in range(width * page)] for b in range(seqs)]

    def more(self):
        """The keyword arguments that a call needs of it."""
        return dict(block_table=self.table, k_scales=self.k_scales, v_scales=self.v_scales)

    def rows(self, which, b, n):
        """What the first n slots of sequence b stand for, [n, heads, 128] in 64 bits on the CPU."""
        pages = torch.tensor([p for p, _ in self.place[b][:n]], dtype=torch.long)
        rows = torch.tensor([r for _, r in self.place[b][:n]], dtype=torch.long)
        cache = getattr(self, which)
        values = cache.view(torch.uint8).cpu()[pages, rows].view(E4M3).double() if n else torch.zeros(0, self.kvh, 128).double()
        return values * self.scales_of(which, b, n)[..., None]

    def scales_of(self, which, b, n):
        """The scales of the first n slots of sequence b, [n, heads] in 64 bits."""
        pages = torch.tensor([p for p, _ in self.place[b][:n]], dtype=torch.long)
        rows = torch.tensor([r for _, r in self.place[b][:n]], dtype=torch.long)
        return getattr(self, which + "_scales").cpu().double()[pages, rows // self.block]

    def snapshot(self):
        return [t.clone() for t in (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scales, self.v_scales)]

    def set(self, which, b, slot, values):
        """Values of a slot, [heads, 128] or what broadcasts to it, as they are in e4m3."""
        page, row = self.place[b][slot]
        cache = getattr(self, which)
        cache.view(torch.uint8)[page, row] = torch.as_tensor(values, dtype=torch.float32).to(E4M3).view(torch.uint8).to(cache.device)


def write(values, scales, first, new, block):
    """What a write of ``new`` [n, 128] (64 bits) from slot ``first`` on makes of one head's e4m3 values [slots, 128] and scales
    [blocks]: new ones of both."""
    values, scales = values.clone(), scales.clone()
    for j in range(first // block, (first + new.size(0) - 1) // block + 1 if new.size(0) else 0):
        lo, hi = max(first, j * block), min(first + new.size(0), (j + 1) * block)
        here = new[lo - first:hi - first]
        finite = here[here.isfinite()].abs()
        most = finite.max().item() if finite.numel() else 0.0
        scale = scale_for(most)
        if lo > j * block:
            had = scales[j].item()
            if most <= 448 * had:
                scale = had
            else:
                values[j * block:lo] = to_e4m3(values[j * block:lo] * (had / scale))
        scales[j] = scale
        values[lo:hi] = torch.where(here.isfinite(), to_e4m3(here / scale), torch.nan)
    return values, scales
