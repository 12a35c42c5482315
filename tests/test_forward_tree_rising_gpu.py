"""Scores that rise steeply at the end of a sequence: a drafted token that attends to itself or its parents above all else, behind many
blocks that the same warps have gone through before.

Tolerance: scores of up to s in 32 bits are off by s 2^-22 or less (128 products, scale), which is the relative error of a
probability; on top of that P's and out's roundings."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import BF16_HALF_STEP, tree_attention
from test_forward_tree_gpu import Batch, visible

pytestmark = pytest.mark.gpu


def raise_scores(batch, slots, factor):
    """K of these slots of every sequence (counted from its first drafted token) along the first query of the sequence's tokens."""
    q = batch.q if not batch.packed else None
    for b, n in enumerate(batch.lens):
        for s, f in zip(slots, factor):
            if 0 <= n + s < n + batch.counts[b]:
                page, row = batch.cache.place[b][n + s]
                batch.cache.k[page, row] = (q[b, max(0, min(s, batch.counts[b] - 1)), :1].float() * f).to(torch.bfloat16)


def check(batch, top):
    out, lse = batch.call()
    min_fa3_op.check_last_status("forward_tree")
    for b in {0, 1, len(batch.lens) // 2, len(batch.lens) - 1}:
        n, c = batch.lens[b], batch.counts[b]
        k, v, seen = batch.cache.rows("k", b, n + c), batch.cache.rows("v", b, n + c), visible(n, c, batch.masks[b])
        ref, ref_lse, _ = tree_attention(batch.q[b].cpu(), k, v, seen)
        size = tree_attention(batch.q[b].cpu(), k, v.abs(), seen)[0]
        assert ((out[b].double().cpu() - ref).abs() <= (BF16_HALF_STEP * 1.1 + top * 2**-21) * (size + ref.abs())).all(), b
        assert (lse[b].double().cpu() - ref_lse).abs().max().item() <= top * 2**-21 + 1e-5, b


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("count", [1, 3, 8, 9, 20, 32, 33, 50, 64, 70, 130])     # of 4 heads: few rows, one tile, two, several items
def test_drafted_tokens_above_all_else(count, tree, seqs=160, length=900):
    """Items of 7 or 8 blocks, about one a CTA, most of them cut once."""
    lens = [length + 13 * b % 101 for b in range(seqs)]
    batch = Batch(count, lens, [count] * seqs, 4, 1, 64, tree=tree)
    raise_scores(batch, range(0, count, 3), [1.0 + 2.0 * i / count for i in range(0, count, 3)])   # 11 to 34 above the others
    check(batch, 100)


@pytest.mark.parametrize("count", [1, 20, 40])
def test_long_items(count):
    """Items of 71 blocks, cut into pieces of a dozen."""
    test_drafted_tokens_above_all_else(count, True, 24, 9000)


@pytest.mark.parametrize("count", [9, 40])
def test_one_row_only(count):
    """The last drafted token alone, so that of a warp's rows one or a few move."""
    batch = Batch(count, [1500 + b for b in range(150)], [count] * 150, 4, 1, 16, tree=False)
    raise_scores(batch, [count - 1], [3.0])
    check(batch, 100)
