"""Values of drafted tokens that are not finite, where a CTA goes through many short items in a row."""
from __future__ import annotations

import pytest
import torch

from test_forward_tree_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [33, 40, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_short_items_of_two_tiles_in_a_row(count, bad):
    """More than 128 rows behind fewer than 128 slots: the block that ends an item is its first or second, so that one tile may be at the
    next item's already when the other asks whether its own had such values."""
    seqs = 600                                                     # four or more items a CTA
    lens = [(37 * b) % 100 for b in range(seqs)]
    batch = Batch(count, lens, [count] * seqs, 4, 1, 16)
    want, want_lse = batch.call()
    sees = torch.zeros(seqs, count, dtype=torch.bool)
    for b in range(0, seqs, 2):                                    # every other one: the items between them have none
        culprit = (7 * b) % count
        page, row = batch.cache.place[b][lens[b] + culprit]
        batch.cache.v[page, row, :, 3:7] = bad
        sees[b] = batch.masks[b][:, culprit]
    assert sees.any() and not sees.all()
    sees = sees.cuda()
    for _ in range(10):
        out, lse = batch.call()
        assert torch.equal(lse, want_lse)
        hit = out[..., 3:7][sees]
        assert (hit.isnan() if bad != bad else hit == bad).all()
        assert torch.equal(out[~sees], want[~sees])
        assert torch.equal(out[..., 7:], want[..., 7:]) and torch.equal(out[..., :3], want[..., :3])
