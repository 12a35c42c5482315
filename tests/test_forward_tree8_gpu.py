"""Attention over a cache in 8 bits against attention in 64 bits over the values that it stands for: trees and chains, head groups,
lengths, caches and scales of every layout, what rows must not see, what has no place, scales far apart, streams and graphs.

Tolerances.  Against 64 bits, a term's probability is rounded to f16: half a step, 2^-11, of it, or half of 2^-24 where f16 has no more
bits, which is 2^-27 of the row's largest term or less.  Scores: Q is off by 2^-18 of a row's largest value where that is
above half of a value's last bit, and products and sums of 128 terms have 32 bits; for scores of a few units 2^-13 of a probability
covers both.  out is rounded to bf16 once.  So |out - ref| <= 2^-8 |ref| + (2^-11 + 2^-12) sum p |v| + floor; and since roundings of
different terms have nothing to do with each other, the 2-norm of the error is at most that of 2^-8 |ref| and 2^-10 times the root of
the terms' squares: a block left out or counted twice would go unnoticed in the first bound, not in this one.  LSE: 2e-5.

The floor: P holds probability times V's scale, its largest in a row at 2^2 or more, and a step of f16 is 2^-24 or more, so a term's
weight is off by 2^-25 / 2^2 = 2^-27 of the row's largest weight at least, times the e4m3 value that it meets: 2^-27 max_s (p_s scale_s)
sum_s |v8_s|.  It is seen where one slot has all the weight and a value of 0."""
from __future__ import annotations

import math
import random

import pytest
import torch

import min_fa3_op
from cache8_util import E4M3, Cache8
from cache_util import BF16_HALF_STEP, ancestors, randn, tree_attention
from test_forward_tree_gpu import visible

pytestmark = pytest.mark.gpu

F16_HALF_STEP = torch.finfo(torch.float16).eps / 2


def floor(q, k, v8, scales, seen):
    """[rows, QH, 128], of the arguments of tree_attention; scales [slots, KVH]."""
    group = q.size(1) // k.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(q.size(0)):
        if not seen[i].any():
            continue
        ki, vi, si = (t[seen[i]].repeat_interleave(group, 1) for t in (k, v8.abs(), scales))
        p = (torch.einsum("hd,shd->hs", q[i].double(), ki) / math.sqrt(128)).softmax(1)
        out[i] = 2**-27 * (p * si.T).amax(1)[:, None] * vi.sum(0)
    return out


class Batch:
    """Queries, cache and masks of one call, and what it has to give."""

    def __init__(self, seed, lens, counts, qh, kvh, page=0, block=16, layout="plain", tree=True, packed=None, slack=0, **more):
        gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.lens, self.counts, self.qh, self.kvh = lens, counts, qh, kvh
        self.cache = Cache8(seed, len(lens), max(n + c for n, c in zip(lens, counts)) + slack, kvh, page, block, layout, **more)
        self.packed = len(set(counts)) > 1 if packed is None else packed
        self.total, self.most = sum(counts), max(counts)
        shape = (self.total,) if self.packed else (len(lens), counts[0])
        self.q = randn(gen, *shape, qh, 128).cuda()
        self.masks = [ancestors(rng, c) if tree else None for c in counts]
        self.tree_mask = None
        if tree:
            rows = torch.zeros(self.total, self.most, dtype=torch.bool)
            first = 0
            for c, m in zip(counts, self.masks):
                rows[first:first + c, :c] = m
                first += c
            self.tree_mask = (rows if self.packed else rows.view(len(lens), self.most, self.most)).cuda()
        self.cu = torch.tensor([0, *torch.tensor(counts).cumsum(0)], dtype=torch.int32).cuda() if self.packed else None
        self.lens_d = torch.tensor(lens, dtype=torch.int32).cuda()

    def call(self, **more):
        args = dict(self.cache.more(), cu_seqlens_q=self.cu, max_seqlen_q=self.most if self.packed else None, tree_mask=self.tree_mask,
                    return_lse=True)
        args.update(more)
        return min_fa3_op.forward_tree(self.q, self.cache.k, self.cache.v, self.lens_d, **args)

    def check(self, out, lse, there=None, scores=0.0):
        """``there``: per sequence the slots that exist.  ``scores``: what scores may be off by beyond what is said above."""
        assert out.is_contiguous() and out.shape == self.q.shape
        q, out = self.q.cpu().reshape(-1, self.qh, 128), out.double().cpu().reshape(-1, self.qh, 128)
        first = 0
        for b, (n, c) in enumerate(zip(self.lens, self.counts)):
            ours_lse = (lse[:, first:first + c] if self.packed else lse[b]).double().cpu()
            k, v = self.cache.rows("k", b, n + c), self.cache.rows("v", b, n + c)
            seen = visible(n, c, self.masks[b])
            if there is not None:
                seen &= there[b]
            ref, ref_lse, spread = tree_attention(q[first:first + c], k, v, seen)
            size = tree_attention(q[first:first + c], k, v.abs(), seen)[0]
            scales = self.cache.scales_of("v", b, n + c)
            least = floor(q[first:first + c], k, v / scales[..., None], scales, seen)
            slack = BF16_HALF_STEP * (1 + 2**-6) * ref.abs() + (F16_HALF_STEP * 1.5 + scores) * size + least + 1e-30
            off = (out[first:first + c] - ref).abs()
            assert (off <= slack).all(), f"sequence {b}: off by {(off / slack).max().item():.2f} of the bound"
            for h in range(self.qh):
                worst = ((BF16_HALF_STEP * ref[:, h].norm()) ** 2 + ((2 * F16_HALF_STEP + scores) * spread[:, h].norm()) ** 2
                         + least[:, h].norm() ** 2).sqrt().item()
                assert off[:, h].norm().item() <= worst + 1e-30, f"sequence {b}, head {h}: {off[:, h].norm().item():.3e} > {worst:.3e}"
            none = torch.isinf(ref_lse)
            assert torch.equal(torch.isinf(ours_lse) & (ours_lse < 0), none)
            if (~none).any():
                assert (ours_lse - ref_lse)[~none].abs().max().item() <= 2e-5 + scores
            first += c


def run(batch, **more):
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    batch.check(out, lse, **more)
    return out, lse


# One sequence, one token; lengths around a block of 128, around two and around the end of a piece; several tiles of rows.
@pytest.mark.parametrize("qh,kvh", [(1, 1), (4, 4), (8, 2), (5, 1), (28, 4), (64, 8), (128, 1)])
@pytest.mark.parametrize("lens,counts", [([0], [1]), ([1], [1]), ([127], [1]), ([128], [1]), ([255], [1]), ([254, 255, 256], [2, 2, 2]),
                                         ([300, 5, 1000], [7, 33, 1])])
def test_head_groups_and_lengths(qh, kvh, lens, counts):
    run(Batch(qh + sum(lens), lens, counts, qh, kvh, page=16, slack=5))


@pytest.mark.parametrize("page,block,layout", [(0, 16, "plain"), (0, 32, "heads"), (0, 128, "layers"), (16, 16, "plain"), (16, 16, "pairs"),
                                               (48, 16, "heads"), (64, 16, "layers"), (64, 64, "pairs"), (96, 32, "plain"),
                                               (128, 128, "pairs"), (160, 32, "plain"), (256, 128, "heads"), (1024, 64, "plain")])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [1, 11, 70])
def test_cache_layouts(page, block, layout, tree, count):
    run(Batch(page + block, [250, 0, 513, 129], [count] * 4, 8, 2, page, block, layout, tree, slack=page // 2))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 63, 64, 65, 130, 300])
def test_numbers_of_drafted_tokens(count, tree):
    run(Batch(count, [200, 77], [count, count], 4, 1, 32, 32, "plain", tree))
    run(Batch(count + 1, [0, 140, 3], [count, 0, max(1, count // 3)], 4, 1, 0, 16, "plain", tree))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("rows", [3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 127, 128, 129, 256, 257])
def test_rows_of_an_item(rows, tree):
    """Where the kernel changes: 4, 8, 16, 32, 128 and 256 rows, one of a token each, and as heads of one token."""
    run(Batch(rows, [0, 200, 1000], [rows, rows, rows // 2], 1, 1, 16, 16, "plain", tree, slack=3))
    if rows <= 128:
        run(Batch(rows, [0, 127, 700], [1, 1, 1], rows, 1, 0, 64, "plain", tree))


@pytest.mark.parametrize("lens,counts,heads", [([20000], [1], (8, 8)), ([20000], [5], (32, 8)), ([9000, 17, 4000, 1], [40, 40, 40, 40], (8, 1)),
                                               ([33000], [70], (8, 1)), ([40000], [2], (4, 1)), ([300] * 150, [2] * 150, (8, 2)),
                                               ([30] * 700, [1] * 700, (2, 1))])
def test_long_caches_and_many_sequences(lens, counts, heads):
    """Items that cross the ends of runs, in two and in many pieces, and runs that cross items and sequences."""
    batch = Batch(len(lens), lens, counts, *heads, page=64)
    out, lse = run(batch)
    junk = torch.empty(64 << 20, device="cuda")
    for fill in range(8):
        junk.fill_(float(fill))                     # the cache is no longer in L2: loads come late, and V later than K
        again = batch.call()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("count,lens", [(1, [3000]), (9, [1500]), (5, [1500]), (40, [900]), (80, [900])])
@pytest.mark.parametrize("slope", [1, -1])
def test_scores_that_rise_and_fall(count, lens, slope):
    """Scores of up to 70, block by block: references move again and again, or lie far above all but the first blocks."""
    batch = Batch(count, lens, [count], 4, 1, 16, tree=False)
    n = lens[0] + count
    ramp = torch.linspace(0.1, 1.0, n)
    if slope < 0:
        ramp = ramp.flip(0)
    direction = batch.q[0, 0, 0].float().cpu()
    direction = direction / direction.abs().max()
    for s in range(n):
        batch.cache.set("k", 0, s, direction * ramp[s] * 448)
    batch.cache.k_scales.fill_(0.03)
    # Scores of up to 70 in 32 bits, 2^-22 of them, and of q 2^-18 of the largest value times the same sum: 70 * 2^-18 in all.
    run(batch, scores=70 * 2**-18)


@pytest.mark.parametrize("count", [1, 8, 40])
def test_a_heavy_slot_and_many_light_ones(count):
    """The first slot has a score 12 above all others, as the first token of a text often has, and they still have a sixth of the
    sum: each of them is 2^-17 of it, and none of that may be lost."""
    batch = Batch(1, [30000 - count], [count], 4, 1, 64, tree=False)
    batch.cache.k.view(torch.uint8).zero_()
    q = batch.q[0].float().cpu()
    batch.q.copy_(batch.q[:, :1, :1].expand_as(batch.q))
    direction = q[0, 0]
    norm = (direction * direction).sum().item()
    batch.cache.set("k", 0, 0, direction)
    page, row = batch.cache.place[0][0]
    got = batch.cache.k.view(torch.uint8)[page, row, 0].cpu().view(E4M3).float()
    batch.cache.k_scales[page, row // 16] = 12 * math.sqrt(128) / (got * direction).sum().item()
    assert norm > 0
    run(batch)


def test_rows_that_see_nothing():
    batch = Batch(10, [0, 5, 0], [6, 6, 6], 8, 2, 16)
    for b, i in ((0, 0), (0, 5), (1, 2), (2, 3)):
        batch.masks[b][i] = False
        batch.tree_mask[b, i] = False
    out, lse = run(batch)
    assert not out[0, 0].any() and torch.isinf(lse[0, :, 0]).all() and torch.isfinite(lse[1, :, 2]).all()


@pytest.mark.parametrize("count,lens", [(1, [70]), (6, [70]), (40, [100]), (150, [0])])
def test_what_a_row_does_not_see_has_no_part(count, lens):
    """Slots behind the last token hold NaN, and so do their blocks' scales; drafted tokens of other branches hold NaN."""
    batch = Batch(count, lens, [count], 4, 1, 16, slack=200)
    n = lens[0]
    want, want_lse = run(batch)
    for s in range(n + count, batch.cache.slots):
        batch.cache.set("k", 0, s, math.nan)
        batch.cache.set("v", 0, s, math.nan)
    for s in range(-(-(n + count) // 16) * 16, batch.cache.slots, 16):
        page, row = batch.cache.place[0][s]
        for scales in (batch.cache.k_scales, batch.cache.v_scales):
            scales[page, row // 16] = [math.nan, math.inf, 0.0, -1.0][s // 16 % 4]
    out, lse = batch.call()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    if count == 1:
        return
    culprit = count // 2                                       # drafted; its descendants see it, the others do not
    sees = batch.masks[0][:, culprit]
    assert sees.any() and not sees.all()
    page, row = batch.cache.place[0][n + culprit]
    keep = batch.cache.v.view(torch.uint8)[page, row].clone()
    batch.cache.v.view(torch.uint8)[page, row, :, 3:7] = 0xFF
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    assert torch.equal(lse, want_lse)
    assert torch.equal(out[0][~sees], want[0][~sees])
    assert torch.equal(out[0][sees][..., 7:], want[0][sees][..., 7:]) and torch.equal(out[0][sees][..., :3], want[0][sees][..., :3])
    assert out[0][sees][..., 3:7].isnan().all()
    batch.cache.v.view(torch.uint8)[page, row] = keep
    batch.cache.set("k", 0, n + culprit, math.nan)
    out, lse = batch.call()
    assert torch.equal(out[0][~sees], want[0][~sees]) and torch.equal(lse[0][:, ~sees], want_lse[0][:, ~sees])
    assert out[0][sees].isnan().all() and lse[0][:, sees].isnan().all()


@pytest.mark.parametrize("count", [20, 5])
def test_nan_in_a_cut_item(count):
    batch = Batch(11, [15000], [count], 4, 1, 64)
    want, _ = run(batch)
    culprit = count // 2
    sees = batch.masks[0][:, culprit]
    page, row = batch.cache.place[0][15000 + culprit]
    batch.cache.v.view(torch.uint8)[page, row, 0, 100] = 0x7F
    out, _ = batch.call()
    assert out[0][sees][..., 100].isnan().all()
    out[..., 100], want[..., 100] = 0, 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("count", [1, 9, 40])
def test_queries_that_are_not_finite(bad, count):
    batch = Batch(12, [300], [count], 4, 1, 16, tree=False)
    want, want_lse = run(batch)
    batch.q[0, count // 2, 1, 77] = bad
    out, lse = batch.call()
    assert out[0, count // 2, 1].isnan().all() and lse[0, 1, count // 2].isnan()
    out[0, count // 2, 1], lse[0, 1, count // 2] = want[0, count // 2, 1], want_lse[0, 1, count // 2]
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("powers", [False, True])
@pytest.mark.parametrize("spread", [0, 12, 40])
@pytest.mark.parametrize("count", [1, 7, 30, 70])
def test_scales_far_apart(spread, powers, count):
    """Scales of blocks between 2^-27 and 2^13.  K: a block of large scores has all the weight.  V: terms that are small relative to the
    largest are off by more of themselves, and by no more of the largest."""
    batch = Batch(spread + count, [700], [count], 8, 2, 32, 16, spread=spread, powers=powers)
    gen = torch.Generator().manual_seed(1)
    batch.cache.k_scales.copy_(torch.exp2(torch.rand(batch.cache.k_scales.shape, generator=gen) * 3 - 9))
    run(batch)
    if spread == 12:
        batch.cache.k_scales.copy_(torch.exp2(torch.rand(batch.cache.k_scales.shape, generator=gen) * spread - 14))
        # Scores of up to 300 in 32 bits, and of q: 300 * 2^-18.
        run(batch, scores=300 * 2**-18)


@pytest.mark.parametrize("count", [1, 40])
def test_expanded_scales(count):
    """One scale for all blocks, or for all heads, expanded."""
    batch = Batch(5, [400, 90], [count] * 2, 8, 2, 64, 32)
    want = dict(batch.cache.more())
    for shape in ((1, 1, 1), (want["k_scales"].size(0), 1, 1), (1, 1, 2)):
        full = want["k_scales"].shape
        batch.cache.k_scales = (torch.rand(shape) * 0.01 + 0.01).cuda().expand(full)
        batch.cache.v_scales = (torch.rand(shape) + 0.5).cuda().expand(full)
        run(batch)


def test_rows_of_zeros_and_of_tiny_and_large_values():
    batch = Batch(6, [300], [8], 4, 1, 16)
    batch.q[0, 1] = 0
    batch.q[0, 2] *= 2.0**-120
    batch.q[0, 3] *= 2.0**-100
    batch.q[0, 4, :, 5:] *= 2.0**-12                  # one value far above the others
    run(batch)
    many = Batch(6, [300], [50], 4, 1, 16)
    many.q[0, 1] = 0
    many.q[0, 2] *= 2.0**-120
    run(many)


@pytest.mark.parametrize("how", ["negative", "behind", "lowest"])
@pytest.mark.parametrize("count", [1, 6, 40, 90])
def test_missing_pages(how, count):
    batch = Batch(8, [500, 300], [count] * 2, 4, 1, 32, 16)
    there = [torch.ones(n + count, dtype=torch.bool) for n in batch.lens]
    for b, entry in ((0, 3), (0, 4), (1, 0), (1, 9)):
        batch.cache.table[b, entry] = {"negative": -1, "behind": batch.cache.k.size(0), "lowest": -2**31}[how]
        there[b][entry * 32:(entry + 1) * 32] = False
    out, lse = batch.call()
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("forward_tree")
    batch.check(out, lse, there=there)


@pytest.mark.parametrize("what", ["beyond the slots", "negative length", "order", "behind the batch"])
def test_lengths_that_do_not_fit_are_reported(what):
    batch = Batch(9, [40, 60, 20], [3, 5, 4], 4, 2, 16)
    if what == "beyond the slots":
        batch.lens_d[1] = batch.cache.slots
    elif what == "negative length":
        batch.lens_d[1] = -7
    else:
        batch.cu[2] = 2 if what == "order" else 100
    out, lse = batch.call()
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("forward_tree")
    first = batch.q.cpu()[:3]
    ref, _, _ = tree_attention(first, batch.cache.rows("k", 0, 43), batch.cache.rows("v", 0, 43), visible(40, 3, batch.masks[0]))
    assert (out[:3].double().cpu() - ref).abs().max().item() <= 2**-7 * ref.abs().max().item()


@pytest.mark.parametrize("rows", [(3, 4, 0), (40, 2, 0)])
def test_padding_rows_are_left_as_they_were(rows):
    """A batch padded for a captured graph: rows behind the last sequence are not written."""
    batch = Batch(13, [100, 30, 64], list(rows), 8, 2, 16, packed=True)
    total = batch.total
    batch.q = torch.cat([batch.q, torch.full((7, 8, 128), math.nan, device="cuda", dtype=torch.bfloat16)])
    batch.tree_mask = torch.cat([batch.tree_mask, torch.ones(7, batch.most, dtype=torch.bool, device="cuda")])
    out = torch.full_like(batch.q, 7.0)
    _, lse = batch.call(out=out)
    min_fa3_op.check_last_status("forward_tree")
    assert (out[total:] == 7).all()
    batch.q, out, lse = batch.q[:total], out[:total], lse[:, :total]
    batch.check(out.contiguous(), lse)


def test_strided_queries():
    batch = Batch(14, [200, 333], [4, 4], 8, 2, 32, 32)
    batch.q = torch.randn(2, 4, 14, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)[:, :, 3:11]
    run(batch)
    many = Batch(15, [200, 333], [50, 50], 8, 2, 32, 32)
    many.q = torch.randn(2, 50, 14, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)[:, :, 3:11]
    run(many)


@pytest.mark.parametrize("count", [1, 9, 80])
def test_captured_and_replayed(count):
    """Lengths, contents, scales and queries change between replays; two captured calls share nothing that one may spoil."""
    one, two = (Batch(seed, [600, 90], [count] * 2, 8, 2, 64, 16, slack=300) for seed in (16, 17))
    for batch in (one, two):
        batch.call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    for batch in (one, two):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            results.append(batch.call())
        graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        for batch in (one, two):
            batch.lens = [n + 70 for n in batch.lens]
            batch.lens_d.add_(70)
            batch.q.copy_(torch.randn_like(batch.q, dtype=torch.float32))
            batch.cache.v_scales.mul_(1.5)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for batch, (out, lse) in zip((one, two), results):
            batch.check(out, lse)


def test_on_another_stream_at_the_same_time():
    big, small = Batch(18, [20000], [2], 8, 2, 64), Batch(19, [900, 33], [60, 60], 8, 2, 16)
    want = [batch.call() for batch in (big, small)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for stream, batch in zip(streams, (big, small)):
            with torch.cuda.stream(stream):
                got.append(batch.call())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_near_the_same_over_a_cache_in_16_bits():
    """Scales that are powers of two: bf16 holds the same values exactly, so the two calls differ by the roundings of both."""
    batch = Batch(20, [700, 64], [6, 6], 8, 2, 64, 32)
    values = [(c.float() * s.repeat_interleave(32, 1)[..., None]).to(torch.bfloat16)
              for c, s in ((batch.cache.k, batch.cache.k_scales), (batch.cache.v, batch.cache.v_scales))]
    out, lse = run(batch)
    wide, wide_lse = min_fa3_op.forward_tree(batch.q, *values, batch.lens_d, block_table=batch.cache.table, tree_mask=batch.tree_mask,
                                             return_lse=True)
    assert (out.float() - wide.float()).norm().item() <= 2**-7 * wide.float().norm().item()
    assert (lse - wide_lse).abs().max().item() <= 3e-5


@pytest.mark.parametrize("count,qh,kvh", [(1, 2, 2), (1, 4, 2), (2, 2, 2), (3, 2, 2), (1, 8, 2), (5, 2, 2), (3, 4, 2), (7, 2, 2), (8, 4, 2)])
@pytest.mark.parametrize("shared", [False, True])
def test_pieces_of_one_block_each_with_its_own_queries(count, qh, kvh, shared):
    """Some hundred sequences of a block or less, so that a CTA's pieces have one block each: 1 to 16 rows, of which some leave a warp
    without any.  ``shared``: all sequences have the same pages, which are at hand, while their queries come from memory."""
    rng = random.Random(count)
    batch = Batch(count, [rng.randint(1, 128 - count) for _ in range(400)], [count] * 400, qh, kvh, 32)
    if shared:
        batch.cache.table.copy_(batch.cache.table[:1].expand_as(batch.cache.table))
        batch.cache.place = [batch.cache.place[0]] * 400
    out, lse = run(batch)
    junk = torch.empty(64 << 20, device="cuda")
    for fill in range(10):
        junk.fill_(float(fill))                     # nothing is in L2 any more; then K, V and their scales, but no queries
        for t in batch.cache.snapshot():
            t.view(torch.uint8).sum()
        again = batch.call()
        min_fa3_op.check_last_status("forward_tree")
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("count", [1, 5, 9, 20, 60, 200])
def test_queries_that_the_two_parts_hold_worst(count):
    """A largest value of 128 and others of 2^-3 + 2^-10, whose rest of 2^-10 lies halfway between two numbers of 8 bits and is lost: 2^-17
    of the largest value in each of 127 terms, all with the same sign.  A row sees its own slot only, so that its lse is the score."""
    batch = Batch(7, [0], [count], 1, 1, 16)
    batch.tree_mask.copy_(torch.eye(count, dtype=torch.bool).view(1, count, count))
    sign = torch.randint(0, 2, (count, 128), generator=torch.Generator().manual_seed(count)) * 2.0 - 1
    q = sign * (2.0**-3 + 2.0**-10)
    q[torch.arange(count), torch.arange(count) % 128] *= 128 / (2.0**-3 + 2.0**-10)
    batch.q.copy_(q.view(1, count, 1, 128))
    assert torch.equal(batch.q.double().cpu().view(count, 128), q.double())
    for s in range(count):
        batch.cache.set("k", 0, s, sign[s] * 448)
    batch.cache.k_scales.fill_(2.0**-9)
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    assert torch.equal(out[0, :, 0].double().cpu(), batch.cache.rows("v", 0, count)[:, 0].to(torch.bfloat16).double())
    score = (q.double() * batch.cache.rows("k", 0, count)[:, 0]).sum(1) / math.sqrt(128)
    off = (lse[0, 0].double().cpu() - score).abs()
    # The 128 terms' roundings, and those of some operations in 32 bits on values of up to the score.
    assert (off <= 2.0**-17 * 128 * 128 * 448 * 2.0**-9 / math.sqrt(128) + 2.0**-20 * score.abs()).all()


@pytest.mark.parametrize("qh,kvh", [(4, 1), (1, 1), (64, 1)])
def test_one_token_with_strides_that_nobody_looks_at(qh, kvh):
    batch = Batch(3, [77], [1], qh, kvh, 16)
    want, want_lse = run(batch)
    batch.q = torch.as_strided(batch.q.clone(), batch.q.shape, (1003, 1001, 5 if qh == 1 else 128, 1))
    out, lse = run(batch)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
