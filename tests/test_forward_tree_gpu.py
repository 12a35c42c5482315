"""Drafted trees over the cache against attention in 64 bits: trees and chains, head groups, lengths, caches of every layout, what
rows must not see, what has no place, streams and graphs.

Tolerances.  Against 64 bits on the same bf16 inputs, out carries the rounding of P (half a step, 2^-8, of each term at most) and
its own (2^-8 of the result): |out - ref| <= 2^-8 (sum p |v| + |ref|), and sums in 32 bits of at most 2^15 terms, whose error is
far below 2^-10 of the same sum.  Roundings of different terms have nothing to do with each other, so over a whole result the
2-norm of the error is at most 2^-8 times that of the root of the terms' squares, and 2^-8 times the result's: a block
left out or counted twice would go unnoticed in the first bound, not in this one.  LSE: scores of a few units in 32 bits, 128 products each, and a sum: 1e-5 covers it."""
from __future__ import annotations

import math
import random

import pytest
import torch

import min_fa3_op
from cache_util import BF16_HALF_STEP, Cache, ancestors, randn, tree_attention

pytestmark = pytest.mark.gpu


def visible(n, count, mask):
    seen = torch.ones(count, n + count, dtype=torch.bool)
    seen[:, n:] = torch.ones(count, count).tril().bool() if mask is None else mask[:count, :count]
    return seen


class Batch:
    """Queries, cache and masks of one call, and what it has to give."""

    def __init__(self, seed, lens, counts, qh, kvh, page=0, layout="plain", tree=True, packed=None, slack=0, scale=1.0):
        gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.lens, self.counts, self.qh, self.kvh = lens, counts, qh, kvh
        self.cache = Cache(seed, len(lens), max(n + c for n, c in zip(lens, counts)) + slack, kvh, page, layout)
        self.packed = len(set(counts)) > 1 if packed is None else packed
        self.total, self.most = sum(counts), max(counts)
        shape = (self.total,) if self.packed else (len(lens), counts[0])
        self.q = (randn(gen, *shape, qh, 128).float() * scale).to(torch.bfloat16).cuda()
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
        args = dict(block_table=self.cache.table, cu_seqlens_q=self.cu, max_seqlen_q=self.most if self.packed else None,
                    tree_mask=self.tree_mask, return_lse=True)
        args.update(more)
        return min_fa3_op.forward_tree(self.q, self.cache.k, self.cache.v, self.lens_d, **args)

    def check(self, out, lse):
        min_fa3_op.check_last_status("forward_tree")
        assert out.is_contiguous() and out.shape == self.q.shape
        q, out = self.q.cpu().reshape(-1, self.qh, 128), out.double().cpu().reshape(-1, self.qh, 128)
        first = 0
        for b, (n, c) in enumerate(zip(self.lens, self.counts)):
            ours_lse = (lse[:, first:first + c] if self.packed else lse[b]).double().cpu()
            k, v = self.cache.rows("k", b, n + c), self.cache.rows("v", b, n + c)
            seen = visible(n, c, self.masks[b])
            ref, ref_lse, spread = tree_attention(q[first:first + c], k, v, seen)
            size = tree_attention(q[first:first + c], k, v.abs(), seen)[0]
            slack = BF16_HALF_STEP * (1 + 2**-4) * (size + ref.abs()) + 1e-30
            off = (out[first:first + c] - ref).abs()
            assert (off <= slack).all(), f"sequence {b}: off by {(off / slack).max().item():.2f} of the bound"
            for h in range(self.qh):
                worst = BF16_HALF_STEP * (spread[:, h].norm() ** 2 + ref[:, h].norm() ** 2).sqrt().item()
                assert off[:, h].norm().item() <= worst + 1e-30, f"sequence {b}, head {h}: {off[:, h].norm().item():.3e} > {worst:.3e}"
            none = torch.isinf(ref_lse)
            assert torch.equal(torch.isinf(ours_lse) & (ours_lse < 0), none)
            if (~none).any():
                assert (ours_lse - ref_lse)[~none].abs().max().item() <= 1e-5
            first += c


# One sequence, one token; lengths around a block of 128 and around the end of a piece; several tiles of rows.
@pytest.mark.parametrize("qh,kvh", [(1, 1), (4, 4), (8, 2), (5, 1), (28, 4), (64, 8), (128, 1)])
@pytest.mark.parametrize("lens,counts", [([0], [1]), ([1], [1]), ([127], [1]), ([128], [1]), ([126, 127, 128], [2, 2, 2]),
                                         ([300, 5, 1000], [7, 33, 1])])
def test_head_groups_and_lengths(qh, kvh, lens, counts):
    batch = Batch(qh + sum(lens), lens, counts, qh, kvh, page=16, slack=5)
    batch.check(*batch.call())


@pytest.mark.parametrize("page,layout", [(0, "plain"), (0, "heads"), (0, "layers"), (8, "plain"), (24, "plain"), (16, "pairs"), (48, "heads"),
                                         (64, "layers"), (128, "pairs"), (160, "plain"), (256, "heads")])
@pytest.mark.parametrize("tree", [False, True])
def test_cache_layouts(page, layout, tree):
    batch = Batch(page, [250, 0, 513, 129], [11, 11, 11, 11], 8, 2, page, layout, tree, slack=page // 2)
    batch.check(*batch.call())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 63, 64, 65, 130, 300])
def test_numbers_of_drafted_tokens(count, tree):
    # 32 tokens of 4 heads are a tile of rows, 64 an item; drafted tokens over several blocks of slots.
    batch = Batch(count, [200, 77], [count, count], 4, 1, 32, "plain", tree)
    batch.check(*batch.call())
    ragged = Batch(count + 1, [0, 140, 3], [count, 0, max(1, count // 3)], 4, 1, 0, "plain", tree)
    ragged.check(*ragged.call())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("rows", [15, 16, 17, 31, 32, 33, 127, 128, 129, 256, 257])
def test_rows_of_an_item(rows, tree):
    """Where the kernel changes: 16, 32, 128 and 256 rows, one of a token each, and as heads of one token."""
    batch = Batch(rows, [0, 200, 1000], [rows, rows, rows // 2], 1, 1, 16, "plain", tree, slack=3)
    batch.check(*batch.call())
    if rows <= 128:
        one = Batch(rows, [0, 127, 700], [1, 1, 1], rows, 1, 0, "plain", tree)
        one.check(*one.call())


@pytest.mark.parametrize("lens,counts,heads", [([20000], [1], (8, 8)), ([20000], [5], (32, 8)), ([9000, 17, 4000, 1], [40, 40, 40, 40], (8, 1)),
                                               ([33000], [70], (8, 1)), ([300] * 150, [2] * 150, (8, 2)), ([30] * 700, [1] * 700, (2, 1))])
def test_long_caches_and_many_sequences(lens, counts, heads):
    """Items that cross the ends of runs, in two and in many pieces, and runs that cross items and sequences."""
    batch = Batch(len(lens), lens, counts, *heads, page=64)
    out, lse = batch.call()
    batch.check(out, lse)
    junk = torch.empty(64 << 20, device="cuda")
    for fill in range(8):
        junk.fill_(float(fill))                     # the cache is no longer in L2: loads come late, and V later than K
        again = batch.call()
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_growing_scores():
    # The running maximum grows from block to block, so that O is scaled again and again.
    batch = Batch(9, [1500], [9], 4, 1, 16, "plain", scale=1.0)
    ramp = torch.linspace(0.2, 12.0, batch.cache.slots).to(torch.bfloat16)
    for s, (page, row) in enumerate(batch.cache.place[0]):
        batch.cache.k[page, row] = (batch.q[0, 0, :1].float() * ramp[s]).to(torch.bfloat16)
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    k, v = batch.cache.rows("k", 0, 1509), batch.cache.rows("v", 0, 1509)
    ref, ref_lse, _ = tree_attention(batch.q[0].cpu(), k, v, visible(1500, 9, batch.masks[0]))
    size = tree_attention(batch.q[0].cpu(), k, v.abs(), visible(1500, 9, batch.masks[0]))[0]
    # Scores of up to 150 in 32 bits: 150 * 2^-22 in the exponent, on top of the two roundings.
    assert ((out[0].double().cpu() - ref).abs() <= (BF16_HALF_STEP * 1.1 + 150 * 2**-21) * (size + ref.abs())).all()
    assert (lse[0].double().cpu() - ref_lse).abs().max().item() <= 150 * 2**-21


@pytest.mark.parametrize("count", [1, 7, 30, 70])
def test_tiny_values(count):
    """V of 2^-70: probabilities are relative to a bound up to 2^32 above some score, so a product may be as small as 2^-102, and
    what is lost below 2^-126 is at most 2^-126 a slot of 2^-32 or more in all: 2^-94 * 240, which is 2^-16 of 2^-70.  Each of the two
    results is rounded once."""
    batch = Batch(count, [210], [count], 4, 1, 16, slack=20)
    want = batch.call()[0].double()
    batch.cache.v *= 2.0**-70
    out = batch.call()[0].double() * 2.0**70
    assert ((out - want).abs() <= 2 * BF16_HALF_STEP * want.abs() + 2**-15).all()


def test_rows_that_see_nothing():
    batch = Batch(10, [0, 5, 0], [6, 6, 6], 8, 2, 16)
    for b, i in ((0, 0), (0, 5), (1, 2), (2, 3)):
        batch.masks[b][i] = False
        batch.tree_mask[b, i] = False
    out, lse = batch.call()
    batch.check(out, lse)
    assert not out[0, 0].any() and torch.isinf(lse[0, :, 0]).all() and torch.isfinite(lse[1, :, 2]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("count,lens", [(6, [70]), (40, [100]), (150, [0])])
def test_what_a_row_does_not_see_has_no_part(bad, count, lens):
    """Slots behind the last token, and drafted tokens of other branches, hold NaN, infinities or the lowest value."""
    heads = (4, 1)
    batch = Batch(count, lens, [count], *heads, 16, slack=60)
    n = lens[0]
    place = batch.cache.place[0]
    for page, row in place[n + count:]:
        batch.cache.k[page, row], batch.cache.v[page, row] = bad, bad
    culprit = count // 2                                       # drafted; its descendants see it, the others do not
    sees = batch.masks[0][:, culprit]
    assert sees.any() and not sees.all()
    want, want_lse = batch.call()
    page, row = place[n + culprit]
    keep_v = batch.cache.v[page, row].clone()
    batch.cache.v[page, row, :, 3:7] = bad
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    assert torch.equal(lse, want_lse)
    assert torch.equal(out[0][~sees], want[0][~sees])
    assert torch.equal(out[0][sees][..., 7:], want[0][sees][..., 7:]) and torch.equal(out[0][sees][..., :3], want[0][sees][..., :3])
    hit = out[0][sees][..., 3:7]
    if math.isfinite(bad):
        batch.check(out, lse)
    else:
        assert (hit.isnan() if math.isnan(bad) else hit == bad).all()
    batch.cache.v[page, row] = keep_v
    batch.cache.k[page, row] = bad if not math.isfinite(bad) else 0.0
    out, lse = batch.call()
    assert torch.equal(out[0][~sees], want[0][~sees]) and torch.equal(lse[0][:, ~sees], want_lse[0][:, ~sees])


def test_not_finite_in_a_cut_item():
    batch = Batch(11, [15000], [20], 4, 1, 64)
    want, _ = batch.call()
    sees = batch.masks[0][:, 8]
    page, row = batch.cache.place[0][15008]
    batch.cache.v[page, row, 0, 100] = float("nan")
    out, _ = batch.call()
    assert out[0][sees][..., 100].isnan().all()
    out[..., 100], want[..., 100] = 0, 0
    assert torch.equal(out, want)


def test_nan_that_a_row_sees_stays():
    batch = Batch(12, [300], [3], 4, 1, 16, tree=False)
    page, row = batch.cache.place[0][10]
    batch.cache.k[page, row] = float("nan")
    out, lse = batch.call()
    assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("view", ["fused", "heads first", "token apart"])
def test_strided_queries_and_masks(view):
    gen = torch.Generator().manual_seed(13)
    batch = Batch(13, [100, 300], [9, 9], 8, 2, 16)
    q = batch.q
    if view == "fused":
        both = torch.cat([randn(gen, 2, 9, 3, 128).cuda(), q, randn(gen, 2, 9, 2, 128).cuda()], 2)
        batch.q = both[:, :, 3:11]
    elif view == "heads first":
        batch.q = q.view(18, 8, 128).transpose(0, 1).contiguous().transpose(0, 1).view(2, 9, 8, 128)
    else:
        batch.q = torch.stack([q, q], 2)[:, :, 0]
    assert torch.equal(batch.q, q)
    wide = torch.ones(2, 12, 40, dtype=torch.bool).cuda()
    wide[:, :9, 5:14] = batch.tree_mask
    batch.check(*batch.call(tree_mask=wide[:, :9, 5:14]))


@pytest.mark.parametrize("count", [1, 6, 40])
def test_pages_that_several_sequences_share(count):
    """A common beginning, stored once, and a page that a sequence's table names twice."""
    batch = Batch(count, [150, 170, 150], [count] * 3, 8, 2, 16)
    for b in (1, 2):
        batch.cache.table[b, :4] = batch.cache.table[0, :4]
        batch.cache.place[b][:64] = batch.cache.place[0][:64]
    batch.cache.table[2, 5] = batch.cache.table[2, 1]
    batch.cache.place[2][80:96] = batch.cache.place[2][16:32]
    batch.check(*batch.call())


def test_out_over_q():
    """out may be q itself: what is read of a row is read before it is written."""
    for count in (1, 9, 60, 150):
        batch = Batch(count, [3000, 40], [count, count], 4, 1, 16)
        want, want_lse = batch.call()
        out, lse = batch.call(out=batch.q)
        assert out is batch.q and torch.equal(out, want) and torch.equal(lse, want_lse)


def test_padded_batch_keeps_the_rows_behind_it():
    batch = Batch(14, [100, 0, 64], [3, 5, 1], 8, 2, 16)
    gen = torch.Generator().manual_seed(14)
    q = torch.cat([batch.q, randn(gen, 7, 8, 128).cuda()])
    mask = torch.cat([batch.tree_mask, torch.ones(7, 5, dtype=torch.bool).cuda()])
    out = torch.full_like(q, 7.0)
    want = batch.call()[0]
    got = batch_call = min_fa3_op.forward_tree(q, batch.cache.k, batch.cache.v, batch.lens_d, block_table=batch.cache.table,
                                               cu_seqlens_q=batch.cu, max_seqlen_q=5, tree_mask=mask, out=out)
    min_fa3_op.check_last_status("forward_tree")
    assert got is out and batch_call is out
    assert torch.equal(out[:9], want) and (out[9:] == 7).all()


@pytest.mark.parametrize("what", ["beyond the slots", "negative length", "page too high", "negative page", "more tokens than said"])
def test_what_does_not_exist_is_reported(what):
    batch = Batch(15, [100, 40], [3, 2], 8, 2, 16)
    want = batch.call()[0]
    if what == "beyond the slots":
        batch.lens_d[1] = batch.cache.slots - 1
    elif what == "negative length":
        batch.lens_d[1] = -5
    elif what == "more tokens than said":
        batch.most = 2
    else:
        batch.cache.table[1, 1] = batch.cache.k.size(0) if what == "page too high" else -1
    out = batch.call()[0]
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("forward_tree")
    if what == "more tokens than said":
        assert torch.equal(out[3:], want[3:])
    else:
        assert torch.equal(out[:3], want[:3])
    ok = Batch(16, [10], [1], 8, 2, 16)
    ok.check(*ok.call())


def test_stream_graph_and_two_graphs():
    """A step captured once serves while lengths, trees and cache change; two graphs replay in turn."""
    first, second = Batch(17, [5000, 9], [4, 4], 8, 2, 16, slack=50), Batch(18, [700], [70], 8, 2, 0, slack=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for b in (first, second):
            b.check(*b.call())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                result = b.call()
            graphs.append((graph, b, result))
    torch.cuda.current_stream().wait_stream(side)
    gen = torch.Generator().manual_seed(19)
    for step in range(3):
        for graph, b, result in graphs:
            b.q.copy_(randn(gen, *b.q.shape))
            b.lens = [n + 7 for n in b.lens]
            b.lens_d.add_(7)
            torch.cuda.synchronize()
        for graph, b, result in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, b, result in graphs:
            eager = b.call()
            b.check(*eager)
            assert torch.equal(result[0], eager[0]) and torch.equal(result[1], eager[1])


def test_equals_the_dense_forward():
    """One token per sequence over equal lengths is what ``forward`` computes."""
    batch = Batch(20, [511] * 3, [1] * 3, 8, 2, 0, tree=False)
    out, lse = batch.call()
    dense, dense_lse = min_fa3_op.forward(batch.q, batch.cache.k[:, :512].contiguous(), batch.cache.v[:, :512].contiguous(), True,
                                          return_lse=True)
    assert (out.float() - dense.float()).abs().max().item() <= 2**-7 * dense.float().abs().max().item()
    assert (lse - dense_lse).abs().max().item() <= 1e-4
