"""Prompts, drafted trees and single tokens with a cache in 8 bits and stretched positions, as a server runs them: writes, attention,
rejected drafts that are written over, blocks whose scale grows.

Each call's attention is held against 64 bits over what the cache then holds, with the tolerances of the tests of ``forward_tree``
over such caches.  What it holds at the end is held against the tokens that were kept.  A value x is rounded to e4m3 when it is written
(2^-4 of it, or half of 2^-9 scales where it is small), and again each time that its block's scale grows, by a power of two, which is
exact except where it is small: half of 2^-9 of the scale then, and the scales that a token has seen, each twice the one before or more,
sum up to twice the last at most.  So it is within 2^-4 |x| + 2 * 2^-10 scale, and 2^-20 of the largest for the turning, as in the tests
of ``rotary``."""
from __future__ import annotations

import math
import random

import pytest
import torch

import min_fa3_op
from cache8_util import E4M3_HALF_STEP, E4M3_SMALLEST, Cache8
from cache_util import randn, turn
from test_forward_tree8_gpu import Batch, run

pytestmark = pytest.mark.gpu

AXES = min_fa3_op.RotaryAxes.from_sections((64,), 1e6).stretched(4, 4096)
FREQ = [(f if keep == 1 else f / 4 + keep * (f - f / 4)) for f, keep in
        ((1e6 ** (-i / 64), min(1.0, max(0.0, (4096 * 1e6 ** (-i / 64) / 6.283185307179586 - 1) / 31))) for i in range(64))]


def turned(x, positions):
    return turn(x.cpu(), positions.cpu()[None], FREQ, [0] * 64, False) * AXES.magnitude


class Server:
    def __init__(self, seed, seqs, qh, kvh, slots, page, block, layout):
        self.gen, self.rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.qh, self.kvh, self.seqs = qh, kvh, seqs
        self.cache = Cache8(seed, seqs, slots, kvh, page, block, layout)
        self.lens = [0] * seqs
        self.kept = [(torch.zeros(0, kvh, 128).double(), torch.zeros(0, kvh, 128).double()) for _ in range(seqs)]
        self.calls = 0

    def tokens(self, total, size):
        q = randn(self.gen, total, self.qh, 128)
        k, v = ((randn(self.gen, total, self.kvh, 128) * size).to(torch.bfloat16) for _ in range(2))
        return q, k, v

    def append(self, counts, positions, q, k, v):
        cu = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
        out = min_fa3_op.append_cache(k.cuda(), v.cuda(), self.cache.k, self.cache.v, torch.tensor(self.lens, dtype=torch.int32).cuda(),
                                      cu_seqlens=cu, q=None if q is None else q.cuda(), positions=positions[None].cuda(), axes=AXES,
                                      **self.cache.more())
        min_fa3_op.check_last_status("append_cache")
        return out

    def attend(self, counts, q, tree):
        self.calls += 1
        batch = Batch(self.calls, self.lens, counts, self.qh, self.kvh, tree=tree, packed=True)
        batch.cache, batch.q = self.cache, q
        # Keys of 12 times the usual size make scores of 60, not of a few units: Q is off by 2^-18 of a row's largest value in each of
        # a product's 128 terms, and those and their sum by 2^-22 in 32 bits.
        sizes = [self.cache.rows("k", b, n + c).abs().sum(2).max().item() for b, (n, c) in enumerate(zip(self.lens, counts))]
        run(batch, scores=(2**-18 + 2**-22) * q.abs().max().item() * max(sizes) / math.sqrt(128))
        return batch.masks

    def keep(self, counts, positions, k, v):
        first, k = 0, turned(k, positions)
        for b, n in enumerate(counts):
            self.kept[b] = tuple(torch.cat([old, new[first:first + n].double()]) for old, new in zip(self.kept[b], (k, v)))
            self.lens[b] += n
            first += n

    def prompt(self, counts):
        q, k, v = self.tokens(sum(counts), 1)
        positions = torch.cat([torch.arange(n, n + c) for n, c in zip(self.lens, counts)])
        self.attend(counts, self.append(counts, positions, q, k, v), False)
        self.keep(counts, positions, k, v)

    def draft(self, counts, size):
        q, k, v = self.tokens(sum(counts), size)
        # Positions by depth come with the masks, which the batch makes from its number: the same ones here.
        masks = Batch(self.calls + 1, self.lens, counts, 1, 1, tree=True, packed=True).masks
        positions = torch.cat([m.sum(1) - 1 + n for n, m in zip(self.lens, masks)])
        self.attend(counts, self.append(counts, positions, q, k, v), True)
        # A path of each tree is kept and written over the first drafted slots, the rest is rejected.
        rows, kept, first = [], [], 0
        for c, m in zip(counts, masks):
            path = m[self.rng.randrange(c)].nonzero()[:, 0].tolist()
            rows += [first + i for i in path]
            kept.append(len(path))
            first += c
        assert self.append(kept, positions[rows], None, k[rows], v[rows]) is None
        self.keep(kept, positions[rows], k[rows], v[rows])

    def check(self):
        for b, n in enumerate(self.lens):
            for which, x in zip("kv", self.kept[b]):
                assert x.size(0) == n
                scale = self.cache.scales_of(which, b, n)[..., None]
                slack = x.abs() * E4M3_HALF_STEP + scale * E4M3_SMALLEST + 2**-20 * AXES.magnitude * x.abs().max()
                off = (self.cache.rows(which, b, n) - x).abs()
                assert (off <= slack).all(), f"{which} of sequence {b}: off by {(off / slack).max().item():.2f} of the bound"


@pytest.mark.parametrize("page,block,layout,qh,kvh", [(16, 16, "plain", 8, 2), (64, 32, "pairs", 4, 4), (0, 128, "heads", 16, 1),
                                                      (48, 16, "layers", 5, 1)])
def test_prompts_drafts_and_single_tokens(page, block, layout, qh, kvh):
    server = Server(page + block, 3, qh, kvh, 400, page, block, layout)
    server.prompt([70, 33, 1])
    server.prompt([1, 64, 130])
    for step in range(6):
        server.draft([5, 1, 9], 1.5**step)
    server.draft([40, 17, 33], 12)
    for step in range(3):
        server.prompt([1, 1, 1])
    server.check()


def test_captured_decoding():
    """One graph of a step: write, attention, lengths and positions go on.  Replayed, and beside it another server's graph on another
    stream; both against the same steps without graphs."""
    def make(seed):
        gen = torch.Generator().manual_seed(seed)
        cache = Cache8(seed, 2, 200, 2, 16, 16)
        data = dict(q=randn(gen, 6, 2, 1, 8, 128).cuda(), k=randn(gen, 6, 2, 1, 2, 128).cuda(), v=randn(gen, 6, 2, 1, 2, 128).cuda())
        return cache, data, torch.tensor([30, 95], dtype=torch.int32).cuda()

    def step(cache, q, k, v, lens):
        turned_q = min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, q=q, positions=lens[None, :, None], axes=AXES, **cache.more())
        return min_fa3_op.forward_tree(turned_q, cache.k, cache.v, lens, **cache.more())

    want = []
    for seed in (1, 2):
        cache, data, lens = make(seed)
        want.append(([], cache))
        for i in range(6):
            want[-1][0].append(step(cache, data["q"][i], data["k"][i], data["v"][i], lens).clone())
            lens += 1
    servers = []
    for seed in (1, 2):
        cache, data, lens = make(seed)
        now = {name: t[0].clone() for name, t in data.items()}
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            out = step(cache, now["q"], now["k"], now["v"], lens)
            lens += 1
        servers.append((cache, data, now, stream, graph, out))
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(6):
        for n, (cache, data, now, stream, graph, out) in enumerate(servers):
            with torch.cuda.stream(stream):
                for name, t in data.items():
                    now[name].copy_(t[i])
                graph.replay()
                got[n].append(out.clone())
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[n], want[n][0]))
        assert all(torch.equal(a, b) for a, b in zip(servers[n][0].snapshot(), want[n][1].snapshot()))


def test_calls_at_once_on_streams_of_their_own():
    """Writes of two caches at the same time, while a third one is read."""
    gen = torch.Generator().manual_seed(9)
    caches = [Cache8(seed, 4, 1200, 2, 16, 16) for seed in (1, 2)]
    k, v = randn(gen, 4, 900, 2, 128).cuda(), randn(gen, 4, 900, 2, 128).cuda()
    lens = torch.tensor([0, 7, 200, 300], dtype=torch.int32).cuda()
    reading = Batch(3, [3000], [4], 8, 2, 64)
    want_out = reading.call()[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for cache, stream in zip(caches, streams):
            with torch.cuda.stream(stream):
                min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, **cache.more())
        with torch.cuda.stream(streams[2]):
            out = reading.call()[0]
    torch.cuda.synchronize()
    assert torch.equal(out, want_out)
    for seed, cache in zip((1, 2), caches):
        alone = Cache8(seed, 4, 1200, 2, 16, 16)
        for _ in range(3):
            min_fa3_op.append_cache(k, v, alone.k, alone.v, lens, **alone.more())
        assert all(torch.equal(a, b) for a, b in zip(cache.snapshot(), alone.snapshot()))


def test_pages_beyond_32_bits():
    """The same step in a cache of 3 pages and in one of 66,000 (4.3 GB each of K and V), on its last ones: the same bits."""
    gen = torch.Generator().manual_seed(10)
    q, k, v = (randn(gen, 1, 150, h, 128).cuda() for h in (8, 8, 8))
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    results = []
    for pages in (3, 66000):
        k_cache, v_cache = (torch.empty(pages, 64, 8, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
        k_scales, v_scales = (torch.empty(pages, 4, 8, device="cuda") for _ in range(2))
        more = dict(block_table=torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda"), k_scales=k_scales,
                    v_scales=v_scales)
        min_fa3_op.append_cache(k, v, k_cache, v_cache, lens, **more)
        min_fa3_op.check_last_status("append_cache")
        results.append(min_fa3_op.forward_tree(q, k_cache, v_cache, lens, return_lse=True, **more))
        results[-1] += (min_fa3_op.forward_tree(q[:, :1], k_cache, v_cache, lens + 149, **more),)
        min_fa3_op.check_last_status("forward_tree")
        del k_cache, v_cache
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_a_prefix_shared_by_pages():
    """Sequences that read the same full pages and go on in pages of their own, against each of them alone."""
    gen = torch.Generator().manual_seed(11)
    cache = Cache8(11, 1, 64 * 8, 2, 64, 16)
    pages = cache.table[0].tolist()
    table = torch.tensor([pages[:2] + [pages[2 + b]] for b in range(4)], dtype=torch.int32).cuda()
    q, k, v = (randn(gen, 4, 5, h, 128).cuda() for h in (8, 2, 2))
    lens = torch.full((4,), 128, dtype=torch.int32, device="cuda")
    scales = dict(k_scales=cache.k_scales, v_scales=cache.v_scales)
    before = cache.snapshot()
    min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, block_table=table, **scales)
    out = min_fa3_op.forward_tree(q, cache.k, cache.v, lens, block_table=table, **scales)
    for b in range(4):
        one = dict(scales, block_table=table[b:b + 1])
        alone = min_fa3_op.forward_tree(q[b:b + 1], cache.k, cache.v, lens[:1], **one)
        assert (out[b:b + 1].float() - alone.float()).abs().max().item() <= 2**-7 * alone.float().abs().max().item()
    for old, new in zip(before, cache.snapshot()):
        assert torch.equal(old[pages[:2]], new[pages[:2]])
