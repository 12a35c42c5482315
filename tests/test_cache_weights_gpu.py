"""Attention weights that cache slots received, against 64 bits.

Tolerance: a score of a few units from 128 products in 32 bits is off by less than 1e-5, which is the relative error of its
exponential; the exponential itself and the scaled lse add 2^-21; sums in 32 bits of up to some thousand positive terms 2^-18."""
from __future__ import annotations

import math

import pytest
import torch

import min_fa3_op
from test_forward_tree_gpu import Batch, visible

pytestmark = pytest.mark.gpu


def reference(batch, lse, weights):
    want = weights.double().cpu().clone()
    q, group = batch.q.cpu().reshape(-1, batch.qh, 128).double(), batch.qh // batch.kvh
    first = 0
    for b, (n, c) in enumerate(zip(batch.lens, batch.counts)):
        k = batch.cache.rows("k", b, n + c).repeat_interleave(group, 1)
        given = (lse[:, first:first + c] if batch.packed else lse[b]).double().cpu()
        s = torch.einsum("thd,shd->hts", q[first:first + c], k) / math.sqrt(128) - given[:, :, None]
        p = torch.where(visible(n, c, batch.masks[b]) & torch.isfinite(given)[:, :, None], s.exp(), 0.0)
        want[b, :, :n + c] += p.view(batch.kvh, group, c, n + c).sum((1, 2))
        first += c
    return want


def call(batch, lse, weights, **more):
    args = dict(block_table=batch.cache.table, cu_seqlens_q=batch.cu, max_seqlen_q=batch.most if batch.packed else None,
                tree_mask=batch.tree_mask)
    args.update(more)
    return min_fa3_op.cache_weights(batch.q, lse, batch.cache.k, batch.lens_d, weights, **args)


def check(batch, start=0.5, lse=None):
    lse = batch.call()[1] if lse is None else lse
    weights = torch.full((len(batch.lens), batch.kvh, batch.cache.slots), start).cuda()
    want = reference(batch, lse, weights)
    before = weights.clone()
    assert call(batch, lse, weights) is weights
    min_fa3_op.check_last_status("cache_weights")
    grown = want - start
    off = (weights.double().cpu() - want).abs()
    assert (off <= 2e-5 * grown + 2**-23 * want.abs()).all(), f"off by {off.max().item():.3e}"
    for b, (n, c) in enumerate(zip(batch.lens, batch.counts)):
        assert torch.equal(weights[b, :, n + c:], before[b, :, n + c:]), "slots behind a sequence changed"
    again = before.clone()
    call(batch, lse, again)
    assert torch.equal(again, weights)
    return weights


@pytest.mark.parametrize("qh,kvh", [(1, 1), (4, 4), (8, 2), (5, 1), (28, 4), (64, 8), (128, 1)])
@pytest.mark.parametrize("lens,counts", [([0], [1]), ([127], [1]), ([126, 127, 128], [2, 2, 2]), ([300, 5, 1000], [7, 33, 1])])
def test_head_groups_and_lengths(qh, kvh, lens, counts):
    check(Batch(qh + sum(lens), lens, counts, qh, kvh, page=16, slack=5))


@pytest.mark.parametrize("page,layout", [(0, "heads"), (0, "layers"), (24, "plain"), (16, "pairs"), (128, "pairs"), (160, "plain")])
@pytest.mark.parametrize("tree", [False, True])
def test_cache_layouts(page, layout, tree):
    check(Batch(page, [250, 0, 513, 129], [11, 11, 11, 11], 8, 2, page, layout, tree, slack=page // 2))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [31, 32, 33, 64, 65, 130, 300])
def test_numbers_of_rows(count, tree):
    # Of 4 heads 32 tokens are a tile; more than 64 go over the slots several times.
    check(Batch(count, [200, 77], [count, count], 4, 1, 32, "plain", tree))
    check(Batch(count + 1, [0, 140, 3], [count, 0, max(1, count // 3)], 4, 1, 0, "plain", tree))


@pytest.mark.parametrize("lens,counts,heads", [([20000], [5], (32, 8)), ([9000, 17, 4000, 1], [40, 40, 40, 40], (8, 1)),
                                               ([33000], [140], (8, 1)), ([300] * 150, [2] * 150, (8, 2))])
def test_long_caches_and_many_sequences(lens, counts, heads):
    check(Batch(len(lens), lens, counts, *heads, page=64))


def test_a_row_gives_one_in_all():
    batch = Batch(21, [3000], [16], 8, 2, 16)
    weights = check(batch, start=0.0)
    assert abs(weights.double().sum().item() - 16 * 8) <= 16 * 8 * 2e-5


def test_rows_left_out_and_rows_that_see_nothing():
    batch = Batch(22, [0, 50], [6, 6], 8, 2, 16)
    batch.masks[0][3] = False
    batch.tree_mask[0, 3] = False
    lse = batch.call()[1]
    assert torch.isinf(lse[0, :, 3]).all()
    lse[1, :, 2] = float("inf")                            # a token that was not accepted
    check(batch, lse=lse)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_row_does_not_see_has_no_part(bad):
    batch = Batch(23, [100], [20], 4, 1, 16, slack=40)
    lse = batch.call()[1]
    weights = torch.zeros(1, 1, batch.cache.slots).cuda()
    want = call(batch, lse, weights).clone()
    for page, row in batch.cache.place[0][120:]:
        batch.cache.k[page, row] = bad
    sees = batch.masks[0][:, 9]
    page, row = batch.cache.place[0][109]
    batch.cache.k[page, row] = bad
    lse[:, :, sees.cuda()] = float("inf")                  # leave out the rows that see it
    got = call(batch, lse, torch.zeros_like(weights))
    fewer = Batch(23, [100], [20], 4, 1, 16, slack=40)     # the same, with a clean slot
    clean = call(fewer, lse, torch.zeros_like(weights))
    assert torch.equal(got[..., :109], clean[..., :109]) and torch.equal(got[..., 110:], clean[..., 110:])
    assert got[0, 0, 109] == 0 and torch.isfinite(want).all()


def test_strided_weights_and_fewer_slots_than_the_cache():
    batch = Batch(24, [100, 300], [9, 9], 8, 2, 16, slack=400)
    lse = batch.call()[1]
    whole = torch.zeros(2, 2, batch.cache.slots).cuda()
    call(batch, lse, whole)
    wide = torch.zeros(2, 5, 2, 400).cuda()
    part = wide[:, 3, :, 20:340]
    call(batch, lse, part)
    min_fa3_op.check_last_status("cache_weights")
    assert torch.equal(part, whole[..., :320])
    part.zero_()
    assert not wide.any()
    call(batch, lse, wide[:, 3, :, 20:300])                # slots 300 to 308 do not fit
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("cache_weights")
    assert not wide[:, 3, :, 300:].any() and torch.equal(wide[0, 3, :, 20:300], whole[0, :, :280])


def test_graph_adds_at_every_replay():
    batch = Batch(25, [500, 9], [4, 4], 8, 2, 16, slack=50)
    lse = batch.call()[1]
    weights = torch.zeros(2, 2, batch.cache.slots).cuda()
    once = call(batch, lse, torch.zeros_like(weights)).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        call(batch, lse, weights)
    torch.cuda.current_stream().wait_stream(side)
    weights.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(weights, (once + once) + once)
