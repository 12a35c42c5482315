"""The cache calls together, as a server makes them: prompts go in by chunks, drafted trees attend and are weighed, accepted tokens are
written again, and sequences that outgrow their budget are cut; each step against 64 bits on what lies in the cache."""
from __future__ import annotations

import math
import random

import pytest
import torch

import min_fa3_op
from cache_util import BF16_HALF_STEP, Cache, ancestors, assert_turned, randn, tree_attention, turn
from test_evict_cache_gpu import order

pytestmark = pytest.mark.gpu

QH, KVH, BUDGET, RECENT = 8, 2, 150, 20
FREQ = [1e6 ** (-i / 64) for i in range(64)]
AXIS = [0] * 16 + [1] * 24 + [2] * 24


class Server:
    """Two sequences on pages of 16 slots; everything that the calls keep on the device, and nothing else."""

    def __init__(self, seed):
        self.gen = torch.Generator().manual_seed(seed)
        self.cache = Cache(seed, 2, 400, KVH, 16, "pairs")
        self.lens = torch.zeros(2, dtype=torch.int32).cuda()
        self.weights = torch.zeros(2, KVH, self.cache.slots).cuda()
        self.axes = min_fa3_op.RotaryAxes(FREQ, AXIS)
        self.seen = [0, 0]                 # tokens so far, evicted ones too: positions go on

    def tokens(self, counts):
        total = sum(counts)
        q, k, v = (randn(self.gen, total, h, 128).cuda() for h in (QH, KVH, KVH))
        cu = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda()
        return q, k, v, cu

    def attend(self, q, k, v, cu, counts, positions, mask):
        """Write, attend, weigh; every result checked."""
        c = self.cache
        common = dict(block_table=c.table)
        turned = min_fa3_op.append_cache(k, v, c.k, c.v, self.lens, cu_seqlens=cu, q=q, positions=positions.cuda(), axes=self.axes, **common)
        flat = turn(q.cpu(), positions, FREQ, AXIS, False)
        assert_turned(turned, q.cpu(), flat, 64)
        rows = None
        if mask is not None:
            rows = torch.zeros(sum(counts), max(counts), dtype=torch.bool)
            first = 0
            for n, m in zip(counts, mask):
                rows[first:first + n, :n] = m
                first += n
            rows = rows.cuda()
        args = dict(cu_seqlens_q=cu, max_seqlen_q=max(counts), tree_mask=rows, **common)
        out, lse = min_fa3_op.forward_tree(turned, c.k, c.v, self.lens, return_lse=True, **args)
        before = self.weights.clone()
        min_fa3_op.cache_weights(turned, lse, c.k, self.lens, self.weights, **args)
        min_fa3_op.check_last_status()
        first = 0
        for b, n in enumerate(counts):
            length = int(self.lens[b])
            keys, values = c.rows("k", b, length + n), c.rows("v", b, length + n)
            assert_turned(keys[length:], k.cpu()[first:first + n], turn(k.cpu()[first:first + n], positions[:, first:first + n], FREQ, AXIS, False), 64)
            assert torch.equal(values[length:], v.cpu()[first:first + n].double())
            seen = torch.ones(n, length + n, dtype=torch.bool)
            seen[:, length:] = torch.ones(n, n).tril().bool() if mask is None else mask[b]
            rows_q = turned.cpu()[first:first + n]
            ref, ref_lse, spread = tree_attention(rows_q, keys, values, seen)
            off = (out.cpu()[first:first + n].double() - ref).norm().item()
            assert off <= BF16_HALF_STEP * (spread.norm() ** 2 + ref.norm() ** 2).sqrt().item()
            assert (lse.cpu()[:, first:first + n].double() - ref_lse).abs().max().item() <= 1e-5
            s = torch.einsum("thd,shd->hts", rows_q.double(), keys.repeat_interleave(QH // KVH, 1)) / math.sqrt(128)
            p = torch.where(seen, (s - lse.cpu()[:, first:first + n].double()[:, :, None]).exp(), 0.0)
            grown = p.view(KVH, QH // KVH, n, length + n).sum((1, 2))
            got = (self.weights[b].cpu().double() - before[b].cpu().double())[:, :length + n]
            # As in the tests of cache_weights, and the rounding of what was there.
            assert ((got - grown).abs() <= 2e-5 * grown + 2**-23 * self.weights[b, :, :length + n].cpu().double()).all()
            first += n
        return out

    def evict(self):
        c = self.cache
        lens = self.lens.tolist()
        old_w = self.weights.cpu()
        old_k, old_v = [c.rows("k", b, n) for b, n in enumerate(lens)], [c.rows("v", b, n) for b, n in enumerate(lens)]
        self.lens, self.weights, index = min_fa3_op.evict_cache(c.k, c.v, self.weights, self.lens, BUDGET, recent=RECENT, block_table=c.table)
        min_fa3_op.check_last_status()
        for b, n in enumerate(lens):
            m = min(n, BUDGET)
            assert int(self.lens[b]) == m
            for h in range(KVH):
                place = order(old_w[b, h].tolist(), n, BUDGET, RECENT)
                assert index[b, h, :m].tolist() == place
                assert torch.equal(c.rows("k", b, m)[:, h], old_k[b][place, h]) and torch.equal(c.rows("v", b, m)[:, h], old_v[b][place, h])
                assert torch.equal(self.weights[b, h, :m].cpu(), old_w[b, h][place])


def positions_of(starts, counts, depth=None):
    at = torch.cat([torch.arange(n) + s if depth is None else depth[b] + s for b, (s, n) in enumerate(zip(starts, counts))])
    return torch.stack([at, at // 3, at % 7]).to(torch.int64)


def test_prompt_drafts_acceptance_and_eviction():
    server, rng = Server(1), random.Random(1)
    for counts in ([100, 37], [61, 130]):                     # prompts, in two chunks each
        q, k, v, cu = server.tokens(counts)
        server.attend(q, k, v, cu, counts, positions_of(server.seen, counts), None)
        server.lens += torch.tensor(counts, dtype=torch.int32).cuda()
        server.seen = [s + n for s, n in zip(server.seen, counts)]
    server.evict()
    for step in range(5):
        counts = [rng.randint(1, 24), rng.randint(1, 40)]     # items of up to 64 rows in some steps, of more in others
        mask = [ancestors(rng, n) for n in counts]
        depth = [m.sum(1) - 1 for m in mask]
        q, k, v, cu = server.tokens(counts)
        positions = positions_of(server.seen, counts, depth)
        server.attend(q, k, v, cu, counts, positions, mask)
        # One path of each tree is accepted: its tokens are written again, in a row this time.
        paths = [torch.nonzero(m[rng.randrange(n)]).flatten() for m, n in zip(mask, counts)]
        keep = torch.cat([p + (0 if b == 0 else counts[0]) for b, p in enumerate(paths)])
        taken = [len(p) for p in paths]
        cu = torch.tensor([0, taken[0], sum(taken)], dtype=torch.int32).cuda()
        min_fa3_op.append_cache(k[keep.cuda()], v[keep.cuda()], server.cache.k, server.cache.v, server.lens, block_table=server.cache.table,
                                cu_seqlens=cu, positions=positions[:, keep].cuda(), axes=server.axes)
        first = 0
        for b, n in enumerate(taken):
            length = int(server.lens[b])
            got = server.cache.rows("k", b, length + n)[length:]
            assert_turned(got, k.cpu()[keep[first:first + n]], turn(k.cpu()[keep[first:first + n]], positions[:, keep[first:first + n]], FREQ, AXIS, False), 64)
            first += n
        server.lens += torch.tensor(taken, dtype=torch.int32).cuda()
        server.seen = [s + n for s, n in zip(server.seen, taken)]
        server.evict()


def test_a_whole_step_in_one_graph():
    """Write, attend, weigh, evict, captured once and replayed over growing sequences, equal to the same calls made one by one."""
    def make():
        gen = torch.Generator().manual_seed(3)
        cache = Cache(5, 3, 96, KVH, 16)
        state = dict(lens=torch.tensor([40, 63, 64], dtype=torch.int32).cuda(), weights=torch.rand(3, KVH, cache.slots, generator=gen).cuda())
        return cache, state
    axes = min_fa3_op.RotaryAxes.from_sections((64,))
    gen = torch.Generator().manual_seed(4)
    inputs = [[randn(gen, 3, 1, h, 128).cuda() for h in (QH, KVH, KVH)] for _ in range(6)]
    q, k, v = (x.clone() for x in inputs[0])
    positions = torch.zeros(1, 3, 1, dtype=torch.int64).cuda()

    def step(cache, lens, weights):
        turned = min_fa3_op.append_cache(k, v, cache.k, cache.v, lens, block_table=cache.table, q=q, positions=positions, axes=axes)
        out, lse = min_fa3_op.forward_tree(turned, cache.k, cache.v, lens, block_table=cache.table, return_lse=True)
        min_fa3_op.cache_weights(turned, lse, cache.k, lens, weights, block_table=cache.table)
        new_lens, new_weights, _ = min_fa3_op.evict_cache(cache.k, cache.v, weights, lens + 1, 64, recent=8, block_table=cache.table)
        lens.copy_(new_lens)
        weights.copy_(new_weights)
        return out

    eager_cache, eager = make()
    wanted = []
    for n, new in enumerate(inputs):
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        positions.fill_(100 + n)
        wanted.append(step(eager_cache, eager["lens"], eager["weights"]).clone())
    cache, state = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = step(cache, state["lens"], state["weights"])
    torch.cuda.current_stream().wait_stream(side)
    for n, new in enumerate(inputs):
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        positions.fill_(100 + n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wanted[n]), n
    assert torch.equal(cache.k, eager_cache.k) and torch.equal(state["weights"], eager["weights"]) and torch.equal(state["lens"], eager["lens"])


def test_two_streams_at_once():
    """Calls on two streams that do not wait for one another, each with its own cache."""
    def batch(seed):
        gen = torch.Generator().manual_seed(seed)
        cache = Cache(seed, 4, 3000, KVH, 16)
        lens = torch.tensor([2900, 17, 1000, 2000], dtype=torch.int32).cuda()
        return cache, lens, randn(gen, 4, 5, QH, 128).cuda()
    work = [batch(11), batch(12)]
    want = [min_fa3_op.forward_tree(q, c.k, c.v, lens, block_table=c.table) for c, lens, q in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(20):
        got = []
        for stream, (c, lens, q) in zip(streams, work):
            with torch.cuda.stream(stream):
                got.append(min_fa3_op.forward_tree(q, c.k, c.v, lens, block_table=c.table))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_pool_of_more_than_2_to_the_31_elements():
    """Pages far behind the first 2^31 values, and 2^32 bytes, of a pool."""
    pages, page = 70000, 128
    pool = torch.zeros(pages, 2, page, KVH, 128, dtype=torch.bfloat16, device="cuda")        # 4.6 billion values, 9.2 GB
    k_cache, v_cache = pool[:, 0], pool[:, 1]
    gen = torch.Generator().manual_seed(6)
    table = torch.tensor([[69999, 3, 40000], [35000, 69998, 0]], dtype=torch.int32).cuda()
    lens = torch.tensor([300, 140], dtype=torch.int32).cuda()
    k, v = randn(gen, 2, 300, KVH, 128).cuda(), randn(gen, 2, 300, KVH, 128).cuda()
    min_fa3_op.append_cache(k, v, k_cache, v_cache, torch.zeros_like(lens), block_table=table)
    q, more_k, more_v = (randn(gen, 2, 3, h, 128).cuda() for h in (QH, KVH, KVH))
    min_fa3_op.append_cache(more_k, more_v, k_cache, v_cache, lens, block_table=table)
    out, lse = min_fa3_op.forward_tree(q, k_cache, v_cache, lens, block_table=table, return_lse=True)
    weights = torch.zeros(2, KVH, 384, device="cuda")
    min_fa3_op.cache_weights(q, lse, k_cache, lens, weights, block_table=table)
    min_fa3_op.check_last_status()
    for b, n in enumerate((300, 140)):
        keys = torch.cat([k[b, :n], more_k[b]]).cpu()
        values = torch.cat([v[b, :n], more_v[b]]).cpu()
        seen = torch.ones(3, n + 3, dtype=torch.bool)
        seen[:, n:] = torch.ones(3, 3).tril().bool()
        ref, ref_lse, spread = tree_attention(q[b].cpu(), keys, values, seen)
        assert (out[b].cpu().double() - ref).norm() <= BF16_HALF_STEP * (spread.norm() ** 2 + ref.norm() ** 2).sqrt()
        assert (lse[b].cpu().double() - ref_lse).abs().max() <= 1e-5
        assert abs(weights[b].sum().item() - 3 * QH) <= 3 * QH * 2e-5
        before = [torch.cat([x[b, :n], y[b]]).cpu() for x, y in ((k, more_k), (v, more_v))]
        after = min_fa3_op.evict_cache(k_cache, v_cache, weights[b:b + 1].contiguous(), lens[b:b + 1] + 3, 100, recent=10,
                                       block_table=table[b:b + 1])
        min_fa3_op.check_last_status()
        at = torch.arange(100)
        pages_of, rows = table[b].cpu().long()[at // page].cuda(), (at % page).cuda()
        for cache, old in ((k_cache, before[0]), (v_cache, before[1])):
            got = cache[pages_of, rows].cpu()
            for h in range(KVH):
                assert torch.equal(got[:, h], old[after[2][0, h].cpu().long(), h])
