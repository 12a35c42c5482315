"""Bounds and sizes at their ends: the largest ``max_seqlen_q``."""
from __future__ import annotations

import pytest
import torch

from test_cache_weights_gpu import call as add_weights
from test_forward_tree_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[2, 1, 5], [1, 90, 0], [200, 3, 300]])
def test_a_loose_bound_on_the_tokens_changes_nothing(counts):
    batch = Batch(sum(counts), [100, 0, 700], counts, 4, 1, 16, tree=False, packed=True)
    out, lse = batch.call()
    weights = add_weights(batch, lse, torch.zeros(3, 1, batch.cache.slots).cuda())
    for most in (max(counts) + 1, 1 << 20, 2**31 - 1):
        loose_out, loose_lse = batch.call(max_seqlen_q=most)
        batch.check(loose_out, loose_lse)
        assert (loose_lse - lse).abs().max().item() <= 1e-5
        loose = add_weights(batch, lse, torch.zeros_like(weights), max_seqlen_q=most)
        assert ((loose - weights).abs() <= 2**-16 * weights).all()
