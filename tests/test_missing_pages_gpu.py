"""Pages that do not exist: their slots take no part in attention and receive none, the rest of the call is right, and it is reported.

Tolerances: those of the tests of ``forward_tree`` and ``cache_weights`` themselves."""
from __future__ import annotations

import math

import pytest
import torch

import min_fa3_op
from cache_util import BF16_HALF_STEP, tree_attention
from test_cache_weights_gpu import call as add_weights
from test_forward_tree_gpu import Batch, visible

pytestmark = pytest.mark.gpu


def check(batch, holes, how):
    """``holes``: (sequence, entry of its table) of pages that do not exist."""
    page = batch.cache.page
    there = [torch.ones(n + c, dtype=torch.bool) for n, c in zip(batch.lens, batch.counts)]
    for b, entry in holes:
        batch.cache.table[b, entry] = {"negative": -1, "behind": batch.cache.k.size(0), "far": 2**31 - 1, "lowest": -2**31}[how]
        there[b][entry * page:(entry + 1) * page] = False
    out, lse = batch.call()
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("forward_tree")
    again = batch.call()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    start = torch.rand(len(batch.lens), batch.kvh, batch.cache.slots, generator=torch.Generator().manual_seed(1)).cuda()
    weights = add_weights(batch, lse, start.clone())
    with pytest.raises(RuntimeError, match="device-side check failed"):
        min_fa3_op.check_last_status("cache_weights")
    q, ours, group, first = batch.q.cpu().reshape(-1, batch.qh, 128), out.double().cpu().reshape(-1, batch.qh, 128), batch.qh // batch.kvh, 0
    for b, (n, c) in enumerate(zip(batch.lens, batch.counts)):
        ours_lse = (lse[:, first:first + c] if batch.packed else lse[b]).double().cpu()
        k, v = batch.cache.rows("k", b, n + c), batch.cache.rows("v", b, n + c)
        seen = visible(n, c, batch.masks[b]) & there[b]
        rows = q[first:first + c]
        ref, ref_lse, _ = tree_attention(rows, k, v, seen)
        size = tree_attention(rows, k, v.abs(), seen)[0]
        slack = BF16_HALF_STEP * (1 + 2**-4) * (size + ref.abs()) + 1e-30
        assert ((ours[first:first + c] - ref).abs() <= slack).all(), f"sequence {b}"
        none = ~seen.any(1)
        assert torch.equal(torch.isinf(ours_lse) & (ours_lse < 0), none.expand(batch.qh, c))
        assert not ours[first:first + c][none].any()
        if not none.all():
            assert (ours_lse - ref_lse)[:, ~none].abs().max().item() <= 1e-5
        s = torch.einsum("thd,shd->hts", rows.double(), k.repeat_interleave(group, 1)) / math.sqrt(128) - ours_lse[:, :, None]
        grown = torch.where(seen & ~none[:, None], s.exp(), 0.0).view(batch.kvh, group, c, n + c).sum((1, 2))
        want, got = start[b, :, :n + c].double().cpu() + grown, weights[b, :, :n + c].double().cpu()
        assert ((got - want).abs() <= 2e-5 * grown + 2**-23 * want.abs()).all(), f"sequence {b}"
        assert torch.equal(weights[b, :, :n + c].cpu()[:, ~there[b]], start[b, :, :n + c].cpu()[:, ~there[b]])
        first += c


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [1, 4, 8, 30, 70])          # of 4 heads: 16 and 32 rows, one tile, two tiles
@pytest.mark.parametrize("page,how", [(16, "negative"), (64, "behind"), (128, "far"), (48, "lowest")])
def test_slots_of_missing_pages_take_no_part(count, page, how, tree):
    lens = [700, 0, 330, 200, 15]
    batch = Batch(count + page, lens, [count] * 5, 4, 1, page, tree=tree)
    last = (200 + count - 1) // page                             # of sequence 3, with its last drafted tokens
    check(batch, [(0, 0), (0, 3), (0, 700 // page), (2, 1), (3, last)], how)


@pytest.mark.parametrize("count", [1, 9, 40])
def test_all_pages_missing_and_items_that_are_cut(count):
    batch = Batch(count, [9000, 100, 300], [count] * 3, 8, 2, 64)
    check(batch, [(0, e) for e in (0, 1, 2, 70, 139)] + [(1, e) for e in range((100 + count - 1) // 64 + 1)], "negative")
    clean = Batch(count, [90, 300], [count] * 2, 8, 2, 64)       # the next call's status is its own
    clean.check(*clean.call())


def test_many_query_rows_go_over_the_slots_several_times():
    batch = Batch(5, [1000, 40], [300, 300], 4, 1, 16, tree=False)
    check(batch, [(0, 2), (0, 61), (0, 70), (1, 0), (1, 1)], "behind")
