"""Partial results in a buffer of their own, and behind the status in one workspace: the same results, and only the status is kept."""
from __future__ import annotations

import pytest
import torch

import min_fa3_op
from cache_util import Cache
from min_fa3_demo_b200 import cache, min_fa3_op as op
from test_forward_tree_gpu import Batch

pytestmark = pytest.mark.gpu


def kept(entry):
    return op._LAST.workspaces[entry].untyped_storage().nbytes()


@pytest.mark.parametrize("count", [1, 8, 9, 32, 33, 70])       # of 4 heads: few rows, one tile, two tiles
def test_forward_tree(monkeypatch, count):
    batch = Batch(count, [9000, 3, 700], [count] * 3, 4, 1, 16)
    out, lse = batch.call()
    batch.check(out, lse)
    assert kept("forward_tree") <= op._SCRATCH_KEPT
    del out, lse
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out, lse = batch.call()
    assert torch.cuda.memory_allocated() - before <= 2 * (out.numel() + lse.numel() * 2) + 4096
    monkeypatch.setattr(cache, "_tree_bytes", lambda lib, index, *sizes: (lib.b2a_tree_fwd_workspace_bytes(*sizes), 0))
    one_out, one_lse = batch.call()
    assert kept("forward_tree") > op._SCRATCH_KEPT and torch.equal(one_out, out) and torch.equal(one_lse, lse)
    min_fa3_op.check_last_status("forward_tree")


@pytest.mark.parametrize("budget,recent", [(1000, 100), (2900, 0), (40, 40)])
def test_evict_cache(monkeypatch, budget, recent):
    def call():
        there = Cache(3, 40, 3000, 2, 16)
        weights = torch.rand(40, 2, there.slots, generator=torch.Generator().manual_seed(1)).cuda()
        lens = (torch.arange(40, dtype=torch.int32) * 75 + 70).cuda()
        result = min_fa3_op.evict_cache(there.k, there.v, weights, lens, budget, recent=recent, block_table=there.table)
        min_fa3_op.check_last_status("evict_cache")
        return (*result, there.k, there.v)
    apart = call()
    assert kept("evict_cache") <= op._SCRATCH_KEPT
    monkeypatch.setattr(cache, "_evict_bytes", lambda lib, *sizes: (lib.b2a_cache_evict_workspace_bytes(*sizes), 0))
    together = call()
    assert all(torch.equal(a, b) for a, b in zip(apart, together))
