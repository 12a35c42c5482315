"""Caches in one piece that are shorter than a block of 128 slots, down to a single slot, and more rows than sequences."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import Cache, randn
from test_cache_weights_gpu import check as check_weights
from test_forward_tree_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["plain", "heads", "layers"])
@pytest.mark.parametrize("lens,count", [([0], 1), ([0, 0, 0], 1), ([3, 0, 6], 1), ([60, 1], 4), ([0, 50], 40), ([20, 56], 70), ([126], 1)])
def test_caches_of_less_than_a_block(lens, count, layout):
    """The box of a load is larger than the cache: what it does not cover reads as zeros and is seen by nobody."""
    batch = Batch(sum(lens) + count, lens, [count] * len(lens), 4, 2, 0, layout)
    assert batch.cache.slots < 128
    batch.check(*batch.call())
    check_weights(batch)


def test_rows_of_the_cache_that_no_sequence_has():
    batch = Batch(7, [40, 5], [3, 3], 4, 2, 0)
    want, want_lse = batch.call()
    junk = torch.full((3, *batch.cache.k.shape[1:]), float("nan"), dtype=torch.bfloat16, device="cuda")
    batch.cache.k, batch.cache.v = torch.cat([batch.cache.k, junk]), torch.cat([batch.cache.v, junk])
    out, lse = batch.call()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_append_and_evict():
    gen = torch.Generator().manual_seed(3)
    cache = Cache(5, 2, 9, 2)
    k, v = randn(gen, 2, 4, 2, 128).cuda(), randn(gen, 2, 4, 2, 128).cuda()
    lens = torch.tensor([5, 0], dtype=torch.int32).cuda()
    min_fa3_op.append_cache(k, v, cache.k, cache.v, lens)
    min_fa3_op.check_last_status("append_cache")
    assert torch.equal(cache.k[0, 5:9], k[0]) and torch.equal(cache.v[1, :4], v[1])
    before = cache.k.clone()
    weights = torch.arange(36, dtype=torch.float32).view(2, 2, 9).flip(-1).contiguous().cuda()
    new, _, index = min_fa3_op.evict_cache(cache.k, cache.v, weights, lens + 4, 6, recent=2)
    min_fa3_op.check_last_status("evict_cache")
    assert new.tolist() == [6, 4] and index[0, 0].tolist() == [0, 1, 2, 3, 7, 8] and index[1, 0].tolist() == [0, 1, 2, 3, -1, -1]
    assert torch.equal(cache.k[0, :6], before[0, index[0, 0].long()]) and torch.equal(cache.k[1], before[1])
